// Rows as 8-bit integers with a scale each: what a product of 8-bit integers reads.
//
//   a = max_c |y[r, c]|     scale[r] = a / 127     q[r, c] = 127 y[r, c] / a, rounded to the nearest integer, ties to even
//
// for y = the row itself; its RMS norm, with the residual's addition in front; or silu(gate) * up.  y is held in 32 bits and
// rounded once, to q.  A row of zeros has the scale 0; a row with an infinity or a NaN has the scale NaN and zeros, so that every
// product with it is NaN.
//
// Plain rows: the quotient is rounded correctly before it is rounded to an integer (Markstein's correction of a product with the
// reciprocal, 1990: r = t - q a exactly by one fused multiply-add, q + r / a), so rows in bfloat16 give the integers of the
// definition, ties included.  The others' y is rounded anyway: one fused multiply-add of y and 127 / a onto a number whose last bit is a
// one gives the integer.  |q| is at most 127.
//
// The large kernels are bounded by memory with the issue slots not far behind (two thirds and three quarters of them used before the
// arithmetic went by pairs), hence pairs of floats, maxima of three and integers in the low bits of floats.
#include <string.h>

#include "nhv_overlap.h"
#include "nhv_vec8.cuh"

namespace {

typedef __nv_bfloat16 bf16;
enum RowKind { ROW_PLAIN = 0, ROW_NORM = 1, ROW_UNIT = 2 };

struct Args {
  int8_t* q;
  float* scales;
  const void* x;
  void* residual;        // ROW_NORM, or null
  const void* weight;    // ROW_NORM
  long long q_stride, x_stride;
  int width;
  float eps, weight_offset;
  int write_residual;
};

__device__ __forceinline__ f32x2 both(float v) { return f2_pack(v, v); }
__device__ __forceinline__ f32x2 f2_add(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// What a row's elements are divided by.  A factor (a power of two) keeps every intermediate of rows of very small and very
// large values in range.
struct Divisor {
  float m, a, inv;       // the factor; the row's largest and its reciprocal, with the factor
};
__device__ __forceinline__ Divisor divisor_of(float a) {
  Divisor d;
  d.m = a < 0x1p-60f ? 0x1p100f : (a > 0x1p100f ? 0x1p-100f : 1.0f);
  d.a = a * d.m;
  d.inv = 1.0f / d.a;
  return d;
}
// 1.5 * 2^23 + q has q's two's complement in its low byte, rounded to nearest, ties to even.
constexpr float LOW_BITS = 12582912.0f;

template <bool EXACT>
__device__ __forceinline__ uint32_t rounded_byte(float y, const Divisor& d) {
  if (!EXACT) return __float_as_uint(fmaf(y * d.m, 127.0f * d.inv, LOW_BITS));
  const float t = y * (127.0f * d.m);
  float q = t * d.inv;
  q = fmaf(fmaf(-q, d.a, t), d.inv, q);
  return __float_as_uint(q + LOW_BITS);
}
__device__ __forceinline__ uint32_t four_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// The special function units.  1 / (1 + e^-g) by them, in units of 2^-24: the exponent of 2, g log2 e, is rounded (1.25 |g|), the exponential is
// within 2^-22 (4), the sum rounds (1), the reciprocal is within an ulp (2).  Below -87.3, where |silu| is less than 2^-119, the reciprocal
// is 0.
__device__ __forceinline__ float exp2_unit(float v) {
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(v));
  return v;
}
__device__ __forceinline__ float reciprocal_unit(float v) {
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(v));
  return v;
}
constexpr float MINUS_LOG2_E = -1.4426950408889634f;

// silu(g) * u.  Rows in 32 bits: within some 5 * 2^-24; gates below -88.7 (|silu| less than 2^-121) give 0.  Rows in 16 bits, whose gates and
// factors have 8: within (9 + 1.25 max(0, -g)) * 2^-24, 34 * 2^-24 for a gate of -20 and 118 for one of -87; the same operations here and by
// pairs in silu_eight, so that a row's integers do not depend on where it lies.
template <typename T> __device__ __forceinline__ float silu_times(float g, float u);
template <> __device__ __forceinline__ float silu_times<float>(float g, float u) { return g / (1.0f + expf(-g)) * u; }
template <> __device__ __forceinline__ float silu_times<bf16>(float g, float u) {
  return g * reciprocal_unit(exp2_unit(g * MINUS_LOG2_E) + 1.0f) * u;
}

// The block's sum and the block's largest magnitude (as the bits of a float that is not negative: their order is that of the
// numbers, with infinities above all numbers and NaN above infinities).  One barrier each; every thread gets the result.
__device__ __forceinline__ float all_sum(float v, float* red) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int n = blockDim.x >> 5;
  float t = (threadIdx.x & 31) < n ? red[threadIdx.x & 31] : 0.f;
  return warp_sum(t);
}
__device__ __forceinline__ uint32_t all_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int n = blockDim.x >> 5;
  return __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < n ? red[threadIdx.x & 31] : 0u);
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// ---------------------------------------------------------------- any width, any alignment
// The row lies in shared memory in 32 bits between the passes (KEEP), or, where it is too long for that, is read again.  One element a thread and
// turn, whatever the address: the norm of 8,192 rows of 5,119 in bfloat16 179 us, of 5,120 the other way 48; plain rows of 24,576 x 4,095 289
// and 47; the unit of 2,048 x 25,601 139 and 46.
constexpr int KEPT_WIDTH = 51200;

template <typename T, int KIND, bool KEEP>
__global__ void rows_kernel(const Args p) {
  extern __shared__ float row[];
  __shared__ float sums[32];
  __shared__ uint32_t tops[32];
  pdl_prologue();
  const long long r = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(p.x) + r * p.x_stride;
  T* residual = KIND == ROW_NORM && p.residual ? reinterpret_cast<T*>(p.residual) + r * (long long)p.width : nullptr;
  const T* w = reinterpret_cast<const T*>(p.weight);
  auto value = [&](int c) -> float {
    if (KIND == ROW_UNIT) return silu_times<T>(to_f32<T>(x[c]), to_f32<T>(x[p.width + c]));
    return to_f32<T>(x[c]);
  };
  uint32_t top = 0;
  if (KIND == ROW_NORM) {
    float ss = 0.f;
    for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
      float s = to_f32<T>(x[c]);
      if (residual) {
        s += to_f32<T>(residual[c]);
        if (p.write_residual) residual[c] = from_f32<T>(s);
      }
      row[c] = s;
      ss = fmaf(s, s, ss);
    }
    const float rstd = 1.0f / sqrtf(all_sum(ss, sums) / (float)p.width + p.eps);
    for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
      const float y = row[c] * rstd * (to_f32<T>(w[c]) + p.weight_offset);
      row[c] = y;
      top = max(top, magnitude(y));
    }
  } else {
    for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
      const float y = value(c);
      if (KEEP) row[c] = y;
      top = max(top, magnitude(y));
    }
  }
  const float a = __uint_as_float(all_max(top, tops));
  const bool finite = a < __int_as_float(0x7f800000), some = finite && a > 0.f;
  if (threadIdx.x == 0) p.scales[r] = finite ? a / 127.0f : __int_as_float(0x7fc00000);
  const Divisor d = divisor_of(some ? a : 1.0f);
  int8_t* q = p.q + r * p.q_stride;
  for (int c = threadIdx.x; c < p.width; c += blockDim.x) q[c] = some ? (int8_t)rounded_byte<KIND == ROW_PLAIN>(KEEP ? row[c] : value(c), d) : (int8_t)0;
}

template <typename T, int KIND>
int launch_any(const Args& p, int n_rows, cudaStream_t stream) {
  int threads = 32;
  while (threads < 1024 && threads * 4 < p.width) threads <<= 1;
  if (p.width > KEPT_WIDTH) {
    if constexpr (KIND == ROW_NORM)
      NHV_REQUIRE(false, "rmsnorm_int8: width %d is beyond the %d floats that a row buffer holds", p.width, KEPT_WIDTH);
    else
      NHV_CUDA(nhv_launch(rows_kernel<T, KIND, false>, dim3(n_rows), dim3(threads), 0, stream, p), "rows_int8");
    return 0;
  }
  static std::atomic<uint64_t> allowed{0};
  NHV_CUDA(nhv_allow_smem((const void*)rows_kernel<T, KIND, true>, KEPT_WIDTH * 4, allowed), "rows_int8");
  NHV_CUDA(nhv_launch(rows_kernel<T, KIND, true>, dim3(n_rows), dim3(threads), (size_t)p.width * 4, stream, p), "rows_int8");
  return 0;
}

// ---------------------------------------------------------------- widths in eights, rows on 16-byte boundaries
// Eight elements as they lie in memory, and as four pairs.
struct Eight {
  f32x2 v[4];
};
template <typename T> struct Piece;
template <> struct Piece<bf16> {
  uint4 v;
  __device__ __forceinline__ void load(const void* row, int i) { v = reinterpret_cast<const uint4*>(row)[i]; }
  __device__ __forceinline__ Eight get() const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    Eight o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.v[i] = f2_pack(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    return o;
  }
};
template <> struct Piece<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const void* row, int i) {
    a = reinterpret_cast<const float4*>(row)[2 * i];
    b = reinterpret_cast<const float4*>(row)[2 * i + 1];
  }
  __device__ __forceinline__ Eight get() const {
    Eight o = {{f2_pack(a.x, a.y), f2_pack(a.z, a.w), f2_pack(b.x, b.y), f2_pack(b.z, b.w)}};
    return o;
  }
};
template <typename T>
__device__ __forceinline__ void store(T* at, const Eight& y) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) f2_unpack(y.v[i], f[2 * i], f[2 * i + 1]);
  nhv_store8(at, f);
}
// max(top, the eight magnitudes); NaN stays
__device__ __forceinline__ void raise_top(float& top, const Eight& y) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    f2_unpack(y.v[i], a, b);
    asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(a), "f"(b));
  }
}
template <typename T>
__device__ __forceinline__ void silu_eight(Eight& g, const Eight& u) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    if (sizeof(T) == 4) {
      float c, d;
      f2_unpack(g.v[i], a, b);
      f2_unpack(u.v[i], c, d);
      g.v[i] = f2_pack(silu_times<float>(a, c), silu_times<float>(b, d));
    } else {                                    // as silu_times<bf16>, by pairs
      f2_unpack(f2_mul(g.v[i], both(MINUS_LOG2_E)), a, b);
      f2_unpack(f2_add(f2_pack(exp2_unit(a), exp2_unit(b)), both(1.0f)), a, b);
      g.v[i] = f2_mul(f2_mul(g.v[i], f2_pack(reciprocal_unit(a), reciprocal_unit(b))), u.v[i]);
    }
  }
}
__device__ __forceinline__ void add_squares(f32x2 (&ss)[2], const Eight& y) {
#pragma unroll
  for (int i = 0; i < 4; ++i) ss[i & 1] = f2_fma(y.v[i], y.v[i], ss[i & 1]);
}
// y * rstd * (w + offset)
__device__ __forceinline__ void scale_eight(Eight& y, Eight w, float rstd, float offset) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (offset != 0.f) w.v[i] = f2_add(w.v[i], both(offset));
    y.v[i] = f2_mul(f2_mul(y.v[i], both(rstd)), w.v[i]);
  }
}
template <bool EXACT>
__device__ __forceinline__ uint2 eight_bytes(Eight y, const Divisor& d) {
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f32x2 z;
    if (EXACT) {
      const f32x2 t = f2_mul(y.v[i], both(127.0f * d.m)), inv = both(d.inv), q = f2_mul(t, inv);
      z = f2_add(f2_fma(f2_fma(q, both(-d.a), t), inv, q), both(LOW_BITS));
    } else {
      if (d.m != 1.0f) y.v[i] = f2_mul(y.v[i], both(d.m));
      z = f2_fma(y.v[i], both(127.0f * d.inv), both(LOW_BITS));
    }
    b[2 * i] = (uint32_t)z;
    b[2 * i + 1] = (uint32_t)(z >> 32);
  }
  return make_uint2(four_bytes(b[0], b[1], b[2], b[3]), four_bytes(b[4], b[5], b[6], b[7]));
}

// A thread keeps CH pieces of its row in registers from the one read to the one write.
template <typename T, int KIND, int CH, int MOST>
__global__ void __launch_bounds__(MOST) rows8_kernel(const Args p) {
  __shared__ float sums[32];
  __shared__ uint32_t tops[32];
  pdl_prologue();
  const long long r = blockIdx.x;
  const int pieces = p.width >> 3;
  const T* x = reinterpret_cast<const T*>(p.x) + r * p.x_stride;
  T* residual = KIND == ROW_NORM && p.residual ? reinterpret_cast<T*>(p.residual) + r * (long long)p.width : nullptr;
  Piece<T> one[CH], two[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c < pieces) {
      one[i].load(x, c);
      if (KIND == ROW_UNIT) two[i].load(x + p.width, c);
      if (KIND == ROW_NORM && residual) two[i].load(residual, c);
    }
  }
  Eight y[CH];
  f32x2 ss[2] = {0ull, 0ull};
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c >= pieces) {
      y[i].v[0] = y[i].v[1] = y[i].v[2] = y[i].v[3] = 0ull;
      continue;
    }
    y[i] = one[i].get();
    if (KIND == ROW_UNIT) silu_eight<T>(y[i], two[i].get());
    if (KIND == ROW_NORM && residual) {
      const Eight u = two[i].get();
#pragma unroll
      for (int e = 0; e < 4; ++e) y[i].v[e] = f2_add(y[i].v[e], u.v[e]);
      if (p.write_residual) store(residual + 8 * c, y[i]);
    }
    if (KIND == ROW_NORM) add_squares(ss, y[i]);
    else raise_top(top, y[i]);
  }
  if (KIND == ROW_NORM) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < pieces) one[i].load(p.weight, c);                  // on its way beside the sum
    }
    const float rstd = 1.0f / sqrtf(all_sum(f2_sum(ss[0], ss[1]), sums) / (float)p.width + p.eps);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      if (threadIdx.x + i * blockDim.x >= pieces) continue;
      scale_eight(y[i], one[i].get(), rstd, p.weight_offset);
      raise_top(top, y[i]);
    }
  }
  const float a = __uint_as_float(all_max(__float_as_uint(top), tops));
  const bool finite = a < __int_as_float(0x7f800000), some = finite && a > 0.f;
  if (threadIdx.x == 0) p.scales[r] = finite ? a / 127.0f : __int_as_float(0x7fc00000);
  const Divisor d = divisor_of(some ? a : 1.0f);
  int8_t* q = p.q + r * p.q_stride;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c < pieces) *reinterpret_cast<uint2*>(q + 8 * c) = some ? eight_bytes<KIND == ROW_PLAIN>(y[i], d) : make_uint2(0, 0);
  }
}

// Wider rows: the row in 32 bits in shared memory, so that two blocks share an SM and one reads while the other writes.
constexpr int WIDE_THREADS = 512;
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}

template <typename T, int KIND>
__global__ void __launch_bounds__(WIDE_THREADS, 2) rows8_wide_kernel(const Args p) {
  extern __shared__ ulonglong2 kept[];           // first and second halves of the eights: neighbouring threads, neighbouring 16 bytes
  __shared__ float sums[32];
  __shared__ uint32_t tops[32];
  pdl_prologue();
  const long long r = blockIdx.x;
  const int pieces = p.width >> 3;
  const T* x = reinterpret_cast<const T*>(p.x) + r * p.x_stride;
  T* residual = KIND == ROW_NORM && p.residual ? reinterpret_cast<T*>(p.residual) + r * (long long)p.width : nullptr;
  f32x2 ss[2] = {0ull, 0ull};
  float top = 0.f;
  const bool pair = KIND == ROW_UNIT || (KIND == ROW_NORM && residual);
  auto keep = [&](int c, const Eight& y) {
    kept[c] = make_ulonglong2(y.v[0], y.v[1]);
    kept[pieces + c] = make_ulonglong2(y.v[2], y.v[3]);
  };
  auto kept_eight = [&](int c) -> Eight {
    const ulonglong2 a = kept[c], b = kept[pieces + c];
    Eight y = {{a.x, a.y, b.x, b.y}};
    return y;
  };
  auto take = [&](int c, const Piece<T>& one, const Piece<T>& two) {
    Eight y = one.get();
    if (KIND == ROW_UNIT) silu_eight<T>(y, two.get());
    if (KIND == ROW_NORM && pair) {
      const Eight u = two.get();
#pragma unroll
      for (int e = 0; e < 4; ++e) y.v[e] = f2_add(y.v[e], u.v[e]);
      if (p.write_residual) store(residual + 8 * c, y);
    }
    if (KIND == ROW_NORM) add_squares(ss, y);
    else raise_top(top, y);
    keep(c, y);
  };
  if (sizeof(T) == 2) {
    // A thread's pieces of both operands lie where its sums will, all of them on their way at once.
    const T* second = KIND == ROW_UNIT ? x + p.width : residual;
    for (int c = threadIdx.x; c < pieces; c += WIDE_THREADS) {
      copy16(&kept[c], x + 8 * c);
      if (pair) copy16(&kept[pieces + c], second + 8 * c);
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
#pragma unroll 2
    for (int c = threadIdx.x; c < pieces; c += WIDE_THREADS) {
      Piece<T> one, two;
      one.load(&kept[c], 0);
      if (pair) two.load(&kept[pieces + c], 0);
      take(c, one, two);
    }
  } else {
    constexpr int CH = 2;
    for (int c0 = threadIdx.x; c0 < pieces; c0 += CH * WIDE_THREADS) {
      Piece<T> one[CH], two[CH];
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = c0 + i * WIDE_THREADS;
        if (c >= pieces) continue;
        one[i].load(x, c);
        if (KIND == ROW_UNIT) two[i].load(x + p.width, c);
        if (KIND == ROW_NORM && residual) two[i].load(residual, c);
      }
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (c0 + i * WIDE_THREADS < pieces) take(c0 + i * WIDE_THREADS, one[i], two[i]);
    }
  }
  if (KIND == ROW_NORM) {
    const float rstd = 1.0f / sqrtf(all_sum(f2_sum(ss[0], ss[1]), sums) / (float)p.width + p.eps);
    for (int c = threadIdx.x; c < pieces; c += WIDE_THREADS) {
      Piece<T> weight;
      weight.load(p.weight, c);
      Eight y = kept_eight(c);
      scale_eight(y, weight.get(), rstd, p.weight_offset);
      raise_top(top, y);
      keep(c, y);
    }
  }
  const float a = __uint_as_float(all_max(__float_as_uint(top), tops));
  const bool finite = a < __int_as_float(0x7f800000), some = finite && a > 0.f;
  if (threadIdx.x == 0) p.scales[r] = finite ? a / 127.0f : __int_as_float(0x7fc00000);
  const Divisor d = divisor_of(some ? a : 1.0f);
  int8_t* q = p.q + r * p.q_stride;
  for (int c = threadIdx.x; c < pieces; c += WIDE_THREADS)
    *reinterpret_cast<uint2*>(q + 8 * c) = some ? eight_bytes<KIND == ROW_PLAIN>(kept_eight(c), d) : make_uint2(0, 0);
}

template <typename T, int KIND, int CH>
int launch_eights(const Args& p, int n_rows, cudaStream_t stream) {
  const int threads = ((p.width / 8 + CH - 1) / CH + 31) / 32 * 32;
  if constexpr (sizeof(T) == 2 || CH > 1) {                       // one piece a thread of 32-bit rows: up to 256 pieces
    if (threads > 256) {
      NHV_CUDA(nhv_launch(rows8_kernel<T, KIND, CH, 1024>, dim3(n_rows), dim3(threads), 0, stream, p), "rows_int8");
      return 0;
    }
  }
  NHV_CUDA(nhv_launch(rows8_kernel<T, KIND, CH, 256>, dim3(n_rows), dim3(threads), 0, stream, p), "rows_int8");
  return 0;
}

// Which kernel and how many pieces a thread; us a call for 1 / 2 / 4 pieces, bfloat16 (before the arithmetic went by pairs, which took a tenth off):
// the norm of 8 rows of 4,096 2.0 / 2.1 / 2.3, of 512 5.3 / 5.8 / 5.5, of 2,048 14.1 / 11.9 / 12.4, of 8,191 of 5,120 64 / 52 / 50; 24,576 plain rows of
// 4,096 74 / 62 / 58; the unit of 8 rows of 12,288 2.8 / 2.7 / 3.0, of 2,048 27.7 / 27.8 / 25.7.  Kept in shared memory / registers: the unit of
// 2,048 rows of 16,384 32 / 34, of 25,600 54 / 74, of 512 rows 17 / 22; of 8,192 rows of 4,096 48 / 30, of 2,048 of 12,288 27 / 25.  In 32 bits the way goes by the
// width alone: it decides in which order a norm's squares are added.
// Now: the norm of 8,191 rows of 5,120 47 us (6.2 TB/s), the unit of 2,048 of 25,600 46 (5.7), 24,576 plain rows of 4,096 47 (6.4), 8 rows of 4,096 1.3 to 2.1.
// In 32 bits the norm of 4,096 rows of 5,120 44 (6.2), the unit of 2,048 of 12,288 55 (4.1: one block of 768 threads an SM), 12,288 plain rows of 4,096 38.
template <typename T, int KIND>
int launch_row(const Args& p, int n_rows, cudaStream_t stream) {
  const long long item = sizeof(T);
  const bool aligned = p.width % 8 == 0 && ((uintptr_t)p.x | (uintptr_t)(p.x_stride * item) | (uintptr_t)(p.width * item) | (uintptr_t)p.residual |
                                            (uintptr_t)p.weight) % 16 == 0 && ((uintptr_t)p.q | (uintptr_t)p.q_stride) % 8 == 0;
  if (!aligned || p.width > KEPT_WIDTH) return launch_any<T, KIND>(p, n_rows, stream);
  const int pieces = p.width / 8;
  if (pieces > (sizeof(T) == 2 && n_rows < 512 ? 4096 : 2047)) {
    static std::atomic<uint64_t> allowed{0};
    NHV_CUDA(nhv_allow_smem((const void*)rows8_wide_kernel<T, KIND>, KEPT_WIDTH * 4, allowed), "rows_int8");
    NHV_CUDA(nhv_launch(rows8_wide_kernel<T, KIND>, dim3(n_rows), dim3(WIDE_THREADS), (size_t)p.width * 4, stream, p), "rows_int8");
    return 0;
  }
  int each = sizeof(T) == 4 ? (pieces <= 256 ? 1 : 2) : n_rows < 1024 ? 1 : KIND == ROW_NORM && pieces <= 512 ? 2 : 4;
  while (each * 1024 < pieces) each *= 2;
  while (each > 1 && pieces <= 32 * (each / 2)) each /= 2;
  if (each == 1) return launch_eights<T, KIND, 1>(p, n_rows, stream);
  if constexpr (sizeof(T) == 2) {                                 // 32-bit rows: up to 2,047 pieces, two a thread
    if (each == 4) return launch_eights<T, KIND, 4>(p, n_rows, stream);
  }
  return launch_eights<T, KIND, 2>(p, n_rows, stream);
}

template <typename T>
int launch_kind(int kind, const Args& p, int n_rows, cudaStream_t stream) {
  if (kind == ROW_PLAIN) return launch_row<T, ROW_PLAIN>(p, n_rows, stream);
  if (kind == ROW_NORM) return launch_row<T, ROW_NORM>(p, n_rows, stream);
  return launch_row<T, ROW_UNIT>(p, n_rows, stream);
}

// ---------------------------------------------------------------- and back
// out[r, c] = q[r, c] * scale[r], in 32 bits, then to out's type.  Bounded by memory: 16 integers a thread where the rows allow it (24,576 rows of 4,096 to
// bfloat16 48 us, 6.2 TB/s).
struct BackArgs {
  const int8_t* q;
  const float* scales;
  void* out;
  long long q_stride, out_stride;
  int n_rows, width;
};

template <typename T>
__global__ void __launch_bounds__(256) values16_kernel(const BackArgs p) {
  pdl_prologue();
  const int pieces = p.width >> 4;
  const long long step = (long long)gridDim.x * 256, all = (long long)p.n_rows * pieces;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += step) {
    const long long r = i / pieces;
    const int c = (int)(i - r * pieces) * 16;
    const uint4 v = *reinterpret_cast<const uint4*>(p.q + r * p.q_stride + c);
    const float s = p.scales[r];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    T* out = reinterpret_cast<T*>(p.out) + r * p.out_stride + c;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (float)(int8_t)(w[2 * h + (e >> 2)] >> (8 * (e & 3))) * s;
      nhv_store8(out + 8 * h, y);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) values_kernel(const BackArgs p) {
  pdl_prologue();
  for (long long r = blockIdx.x; r < p.n_rows; r += gridDim.x) {
    const float s = p.scales[r];
    for (unsigned c = threadIdx.x; c < (unsigned)p.width; c += 256)          // up to 2^31 - 1 columns: the last turn's end has no number in an int
      reinterpret_cast<T*>(p.out)[r * p.out_stride + c] = from_f32<T>((float)p.q[r * p.q_stride + c] * s);
  }
}

template <typename T>
int launch_back(const BackArgs& p, cudaStream_t stream) {
  const bool eights = p.width % 16 == 0 && ((uintptr_t)p.q | (uintptr_t)p.q_stride | (uintptr_t)p.out | (uintptr_t)(p.out_stride * sizeof(T))) % 16 == 0;
  if (eights) {
    const long long blocks = ((long long)p.n_rows * (p.width / 16) + 255) / 256;
    NHV_CUDA(nhv_launch(values16_kernel<T>, dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)), dim3(256), 0, stream, p), "dequantize_rows");
  } else {
    NHV_CUDA(nhv_launch(values_kernel<T>, dim3(p.n_rows), dim3(256), 0, stream, p), "dequantize_rows");
  }
  return 0;
}

}  // namespace

// What a call is given, one after the other, in one block.
struct RowsCall {
  long long q, scales, x, residual, weight, q_stride, x_stride;
  int kind, dtype, n_rows, width, write_residual;
  float eps, weight_offset;
};
static_assert(sizeof(RowsCall) == 88, "the block ends with four bytes that nobody reads");

// kind: 0 the rows of x, 1 their RMS norm (residual may be null), 2 silu(first half) * second half of rows of 2 * width.
NHV_API int nhv_rows_int8(const void* given, cudaStream_t stream) {
  RowsCall c;
  memcpy(&c, given, sizeof(c));
  if (c.n_rows == 0) return 0;
  NHV_REQUIRE(c.n_rows > 0 && c.width > 0 && c.width <= (1 << 30) && c.q && c.scales && c.x, "rows_int8: bad sizes");
  NHV_REQUIRE(c.kind >= ROW_PLAIN && c.kind <= ROW_UNIT && (c.kind != ROW_NORM || c.weight), "rows_int8: bad arguments");
  NHV_REQUIRE(c.dtype == NHV_F32 || c.dtype == NHV_BF16, "rows_int8: unknown dtype %d", c.dtype);
  // A block reads its row while others write theirs: what is written shares no byte with anything else of the call.
  const long long item = c.dtype == NHV_F32 ? 4 : 2, n = c.n_rows, w = c.width;
  const NhvRows q = {c.q, n, c.q_stride, w}, scales = {c.scales, 1, 0, n * 4};
  const NhvRows x = {c.x, n, c.x_stride * item, w * item * (c.kind == ROW_UNIT ? 2 : 1)};
  const NhvRows weight = {c.weight, c.kind == ROW_NORM, 0, w * item}, residual = {c.residual, c.kind == ROW_NORM && c.residual, 0, n * w * item};
  NHV_REQUIRE(!nhv_rows_meet(q, x) && !nhv_rows_meet(q, residual) && !nhv_rows_meet(q, weight) && !nhv_rows_meet(q, scales),
              "the 8-bit rows have memory of their own: other rows are still read from what lies there");
  NHV_REQUIRE(!nhv_rows_meet(scales, x) && !nhv_rows_meet(scales, residual) && !nhv_rows_meet(scales, weight),
              "the scales have memory of their own: other rows are still read from what lies there");
  NHV_REQUIRE(!c.write_residual || (!nhv_rows_meet(residual, x) && !nhv_rows_meet(residual, weight)),
              "the residual has memory of its own: its sum with x is written there");
  const Args p = {(int8_t*)c.q, (float*)c.scales, (const void*)c.x, (void*)c.residual, (const void*)c.weight, c.q_stride, c.x_stride, c.width,
                  c.eps, c.weight_offset, c.write_residual};
  return c.dtype == NHV_F32 ? launch_kind<float>(c.kind, p, c.n_rows, stream) : launch_kind<bf16>(c.kind, p, c.n_rows, stream);
}

struct BackCall {
  long long out, q, scales, out_stride, q_stride;
  int dtype, n_rows, width;
};
static_assert(sizeof(BackCall) == 56, "the block ends with four bytes that nobody reads");

NHV_API int nhv_rows_from_int8(const void* given, cudaStream_t stream) {
  BackCall c;
  memcpy(&c, given, sizeof(c));
  if (c.n_rows == 0 || c.width == 0) return 0;
  NHV_REQUIRE(c.n_rows > 0 && c.width > 0 && c.out && c.q && c.scales && (c.dtype == NHV_F32 || c.dtype == NHV_BF16), "dequantize_rows: bad arguments");
  const NhvRows out = {c.out, c.n_rows, c.out_stride * (c.dtype == NHV_F32 ? 4 : 2), (long long)c.width * (c.dtype == NHV_F32 ? 4 : 2)};
  NHV_REQUIRE(!nhv_rows_meet(out, {c.q, c.n_rows, c.q_stride, c.width}) && !nhv_rows_meet(out, {c.scales, 1, 0, 4LL * c.n_rows}),
              "the values have memory of their own: other rows are still read from what lies there");
  const BackArgs p = {(const int8_t*)c.q, (const float*)c.scales, (void*)c.out, c.q_stride, c.out_stride, c.n_rows, c.width};
  return c.dtype == NHV_F32 ? launch_back<float>(p, stream) : launch_back<bf16>(p, stream);
}
