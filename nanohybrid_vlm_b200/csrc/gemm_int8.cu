// out[t, n] = (sum_k x[t, k] w[n, k]) * x_scales[t] * w_scales[n] for x [T, K] and w [N, K] of 8-bit integers; out bfloat16 or float32.
//
// The sum is exact in 32 bits (K <= 131,071: K * 128 * 128 < 2^31), so no cut of K and no order of adding changes an output: only the
// conversion of the sum to a float and the products with the two scales round, and the store once more.
#include "nhv_common.cuh"

namespace {

typedef __nv_bfloat16 bf16;

struct Product {
  const int8_t *x, *w;
  const float *x_scales, *w_scales;
  void* out;
  long long x_stride, w_stride, out_stride;
  int T, N, K, out_f32;
};

__device__ __forceinline__ float scaled(int sum, float xs, float ws) { return (float)sum * xs * ws; }

__device__ __forceinline__ void store_out(const Product& p, int t, int n, float v) {
  const long long at = (long long)t * p.out_stride + n;
  if (p.out_f32)
    reinterpret_cast<float*>(p.out)[at] = v;
  else
    reinterpret_cast<bf16*>(p.out)[at] = __float2bfloat16_rn(v);
}

// ---------------------------------------------------------------- any size, any alignment
// A tile of 64 x 64 outputs a block, 64 columns of K at a time through shared memory, four products of bytes an instruction.
constexpr int TILE = 64, WORDS = 16;

__device__ __forceinline__ int word_at(const int8_t* row, int k, int K) {
  uint32_t v = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (k + i < K) v |= (uint32_t)(uint8_t)row[k + i] << (8 * i);
  return (int)v;
}

__global__ void __launch_bounds__(256) product_any_kernel(const Product p) {
  __shared__ int xs[TILE][WORDS + 1], ws[TILE][WORDS + 1];
  pdl_prologue();
  const int t0 = blockIdx.y * TILE, n0 = blockIdx.x * TILE, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int sum[4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += 4 * WORDS) {
    __syncthreads();
    for (int i = threadIdx.x; i < TILE * WORDS; i += 256) {
      const int r = i / WORDS, c = i % WORDS;
      xs[r][c] = t0 + r < p.T ? word_at(p.x + (long long)(t0 + r) * p.x_stride, k0 + 4 * c, p.K) : 0;
      ws[r][c] = n0 + r < p.N ? word_at(p.w + (long long)(n0 + r) * p.w_stride, k0 + 4 * c, p.K) : 0;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < WORDS; ++c) {
      int a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = xs[ty + 16 * i][c];
        b[i] = ws[tx + 16 * i][c];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] = __dp4a(a[i], b[j], sum[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = t0 + ty + 16 * i;
    if (t >= p.T) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx + 16 * j;
      if (n < p.N) store_out(p, t, n, scaled(sum[i][j], p.x_scales[t], p.w_scales[n]));
    }
  }
}

}  // namespace

NHV_API int nhv_gemm_int8(void* out, int out_dtype, long long out_stride, const void* x, long long x_stride, const float* x_scales,
                          const void* w, long long w_stride, const float* w_scales, int T, int N, int K, cudaStream_t stream) {
  if (T == 0 || N == 0) return 0;
  NHV_REQUIRE(T > 0 && N > 0 && K > 0 && K <= 131071, "linear_int8: a sum over 1 to 131,071 products is exact in 32 bits, not over %d", K);
  NHV_REQUIRE(out && x && w && x_scales && w_scales && (out_dtype == NHV_F32 || out_dtype == NHV_BF16), "linear_int8: bad arguments");
  const Product p = {(const int8_t*)x, (const int8_t*)w, x_scales, w_scales, out, x_stride, w_stride, out_stride, T, N, K, out_dtype == NHV_F32};
  const int rows = (T + TILE - 1) / TILE;
  NHV_REQUIRE(rows <= 65535, "linear_int8: %d tokens are more than a call takes", T);
  NHV_CUDA(nhv_launch(product_any_kernel, dim3((N + TILE - 1) / TILE, rows), dim3(256), 0, stream, p), "linear_int8");
  return 0;
}
