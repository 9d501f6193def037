// Rows as 8-bit integers with a scale each: what a product of 8-bit integers reads.
//
//   a = max_c |y[r, c]|     scale[r] = a / 127     q[r, c] = 127 y[r, c] / a, rounded to the nearest integer, ties to even
//
// for y = the row itself; its RMS norm, with the residual's addition in front; or silu(gate) * up.  y is held in 32 bits and
// rounded once, to q.  A row of zeros has the scale 0; a row with an infinity or a NaN has the scale NaN and zeros, so that every
// product with it is NaN.
//
// The quotient is rounded correctly before it is rounded to an integer (Markstein's correction of a product with the
// reciprocal, 1990: r = t - q a exactly by one fused multiply-add, q + r / a), so rows in bfloat16 give the integers of the
// definition, ties included.  |q| is at most 127.
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

// What a row's elements are divided by.  The factor m (a power of two) keeps every intermediate of rows of very small and very
// large values in range.
struct Divisor {
  float m, a, inv;
};
__device__ __forceinline__ Divisor divisor_of(float a) {
  Divisor d;
  d.m = a < 0x1p-60f ? 0x1p100f : (a > 0x1p100f ? 0x1p-100f : 1.0f);
  d.a = a * d.m;
  d.inv = 1.0f / d.a;
  return d;
}
// The integer in the low byte: 1.5 * 2^23 + q has q's two's complement there, rounded to nearest, ties to even.
__device__ __forceinline__ uint32_t rounded_byte(float y, const Divisor& d) {
  const float t = y * d.m * 127.0f;
  float q = t * d.inv;
  q = fmaf(fmaf(-q, d.a, t), d.inv, q);
  return __float_as_uint(q + 12582912.0f);
}
__device__ __forceinline__ uint32_t four_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

template <typename T> __device__ __forceinline__ float silu_times(float g, float u);
template <> __device__ __forceinline__ float silu_times<float>(float g, float u) { return g / (1.0f + expf(-g)) * u; }
// Rows in 16 bits: the fast exponential and division, about 2 ulp of 32 bits, next to inputs of 8 bits.
template <> __device__ __forceinline__ float silu_times<bf16>(float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; }

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
// The row lies in shared memory in 32 bits between the passes (KEEP), or, where it is too long for that, is read again.
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
  for (int c = threadIdx.x; c < p.width; c += blockDim.x) q[c] = some ? (int8_t)rounded_byte(KEEP ? row[c] : value(c), d) : (int8_t)0;
}

template <typename T, int KIND>
int launch_any(const Args& p, int n_rows, cudaStream_t stream) {
  int threads = 32;
  while (threads < 1024 && threads * 4 < p.width) threads <<= 1;
  if (p.width <= KEPT_WIDTH) {
    static std::atomic<uint64_t> allowed{0};
    NHV_CUDA(nhv_allow_smem((const void*)rows_kernel<T, KIND, true>, KEPT_WIDTH * 4, allowed), "rows_int8");
    NHV_CUDA(nhv_launch(rows_kernel<T, KIND, true>, dim3(n_rows), dim3(threads), (size_t)p.width * 4, stream, p), "rows_int8");
  } else {
    NHV_REQUIRE(KIND != ROW_NORM, "rmsnorm_int8: width %d is beyond the %d floats that a row buffer holds", p.width, KEPT_WIDTH);
    NHV_CUDA(nhv_launch(rows_kernel<T, KIND == ROW_NORM ? ROW_PLAIN : KIND, false>, dim3(n_rows), dim3(threads), 0, stream, p), "rows_int8");
  }
  return 0;
}

template <typename T>
int launch_kind(int kind, const Args& p, int n_rows, cudaStream_t stream) {
  if (kind == ROW_PLAIN) return launch_any<T, ROW_PLAIN>(p, n_rows, stream);
  if (kind == ROW_NORM) return launch_any<T, ROW_NORM>(p, n_rows, stream);
  return launch_any<T, ROW_UNIT>(p, n_rows, stream);
}

}  // namespace

// kind: 0 the rows of x, 1 their RMS norm (residual may be null), 2 silu(first half) * second half of rows of 2 * width.
NHV_API int nhv_rows_int8(int kind, int dtype, void* q, long long q_stride, float* scales, const void* x, long long x_stride, void* residual,
                          const void* weight, int n_rows, int width, float eps, float weight_offset, int write_residual, cudaStream_t stream) {
  if (n_rows == 0) return 0;
  NHV_REQUIRE(n_rows > 0 && width > 0 && width <= (1 << 30) && q && scales && x, "rows_int8: bad sizes");
  NHV_REQUIRE(kind >= ROW_PLAIN && kind <= ROW_UNIT && (kind != ROW_NORM || weight), "rows_int8: bad arguments");
  NHV_REQUIRE(dtype == NHV_F32 || dtype == NHV_BF16, "rows_int8: unknown dtype %d", dtype);
  const Args p = {(int8_t*)q, scales, x, residual, weight, q_stride, x_stride, width, eps, weight_offset, write_residual};
  return dtype == NHV_F32 ? launch_kind<float>(kind, p, n_rows, stream) : launch_kind<bf16>(kind, p, n_rows, stream);
}
