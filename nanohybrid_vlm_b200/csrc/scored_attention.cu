// Attention over cache pages that also adds up, per cached key, the weight it received: what a cache that is to drop keys
// goes by.  For every new token t of a request (n new ones, L keys in the cache with them) and query head h of KV head g
//   s[j] = cap(scale q . k[j]),  j <= L - n + t;     p[j] = exp(s[j]) / (sum_j exp(s[j]) + exp(sink[h]));     out = sum_j p[j] v[j]
//   scores_out[g][j] = (j < L - n ? scores[g][j] : 0) + sum over t and the heads of g of p[j];     births[g][j] = position, j new
// A key's sum needs the rows' final normaliser, so there are two passes: the rows' (output and log-sum), then the keys'.
//
// The entry point, and kernels for any type, size and page size in 32 bits (the float32 path, and what the tensor-core kernels of
// scored_attention_short.cu and scored_attention_tcgen05.cu refuse).  Products are those of tf32 halves, x y = hi hi + hi lo + lo hi:
// three products of the tensor cores take less than one of the CUDA cores, whose 16-byte reads of shared memory took as long again
// (float32 prompts of 90 to 400 tokens among 400 to 777 keys: 376 us with those, 304 us so, and no less exact).
//   rows: four warps hold 16 rows each (row = token * G + head, of one request and KV head) and walk the keys in tiles of 32 through
//     shared memory; scores stay in registers as the weights of the second product.  Tiles of 32 let three blocks run on an SM (64: two
//     blocks, 236 against 197 us).  A tile's values arrive while its scores are made, the next tile's keys while the values are used.
//   keys: 64 keys stay in shared memory, the tiles of 64 rows pass by; a lane adds up the weights of its 16 keys, the rows' lanes and
//     warps meet at the end.
// What bounds them is the cutting into halves beside the products, with three warps a scheduler: the tensor cores are busy for 36 % of
// the rows' pass and 43 % of the keys', the schedulers for 41 %.
// Long walks over the keys are split over blocks where there are few tiles of rows, and rows into chunks in the keys' pass; two
// small kernels join the parts in a fixed order.  No sum depends on the order in which blocks run.
//
// A key out of sight may hold anything: its score is replaced, and where a tile's sum is not finite its odd values are left out of
// the products and given to the rows that see them.
#include <type_traits>

#include "nhv_scored.cuh"

namespace {

constexpr int SA_THREADS = 128, SA_WARPS = SA_THREADS / 32, SA_ROWS = 16 * SA_WARPS;
constexpr int ROWS_KEYS = 32, KEYS_KEYS = 64;     // keys of a tile in the rows' pass and in the keys' pass

struct TileArgs {
  ScoredArgs a;
  ScoredParts p;
  int vec;                  // rows of q and of the pages can be read four elements at a time
  int vec_out;              // and rows of the output written
};

template <typename T> __device__ __forceinline__ float4 load4(const T* p);
template <> __device__ __forceinline__ float4 load4<float>(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <> __device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}

// ROWS rows of d elements at base + at[r] into shared memory, `stride` floats apart, as fp32, and committed as one group of
// asynchronous copies (float32 rows that can be read by 16 bytes; others are there when this returns).  at[r] < 0: zeros.  The last
// four columns that d reaches into are filled up with zeros.
template <typename T, int DB, int ROWS>
__device__ __forceinline__ void load_rows(float* dst, int stride, const T* base, const long long* at, int d, bool vec) {
  constexpr int PER_ROW = 16 * DB;
#pragma unroll
  for (int i = threadIdx.x; i < ROWS * PER_ROW; i += SA_THREADS) {
    const int r = i / PER_ROW, c = (i - r * PER_ROW) * 4;
    if (c >= d) continue;
    const T* src = base + at[r] + c;
    const bool there = at[r] >= 0;
    if (sizeof(T) == 4 && vec) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"((uint32_t)__cvta_generic_to_shared(dst + r * stride + c)), "l"(there ? src : base),
                   "r"(there ? 16 : 0) : "memory");
      continue;
    }
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (there) {
      if (vec) {
        v = load4<T>(src);
      } else {
        v.x = to_f32<T>(src[0]);
        if (c + 1 < d) v.y = to_f32<T>(src[1]);
        if (c + 2 < d) v.z = to_f32<T>(src[2]);
        if (c + 3 < d) v.w = to_f32<T>(src[3]);
      }
    }
    *reinterpret_cast<float4*>(dst + r * stride + c) = v;
  }
  asm volatile("cp.async.commit_group;\n" ::: "memory");
}
// All groups but the last N have arrived (this thread's copies).
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

// A float32 as two tf32 numbers of 11 bits each: hi its nearest (NEAR: what a row brings) or its first bits (one instruction less: what
// the keys bring; hi lo of one operand that errs to either side leaves no bias), lo what is left of it but for the last bits (3 2^-23
// of x at most).  A bfloat16 is a tf32 as it is.  What is not finite, or rounds to that, gives no finite hi + lo.
struct Halves {
  uint32_t hi, lo;
};
template <bool EXACT, bool NEAR>
__device__ __forceinline__ Halves halves(float x) {
  if (EXACT) return {__float_as_uint(x), 0u};
  const uint32_t hi = (__float_as_uint(x) + (NEAR ? 0x1000u : 0u)) & 0xffffe000u;
  return {hi, __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u};
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// a b[u], u < N, from halves: the products of two upper ones go to c, the small ones to rest.  A_EXACT, B_EXACT: without lower halves.
template <bool A_EXACT, bool B_EXACT, int N>
__device__ __forceinline__ void mma_halves(float (&c)[N][4], float (&rest)[N][4], const Halves (&a)[4], const Halves (&b)[N][2]) {
#pragma unroll
  for (int u = 0; u < N; ++u) mma_tf32(c[u], a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[u][0].hi, b[u][1].hi);
  if (!A_EXACT) {
#pragma unroll
    for (int u = 0; u < N; ++u) mma_tf32(rest[u], a[0].lo, a[1].lo, a[2].lo, a[3].lo, b[u][0].hi, b[u][1].hi);
  }
  if (!B_EXACT) {
#pragma unroll
    for (int u = 0; u < N; ++u) mma_tf32(rest[u], a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[u][0].lo, b[u][1].lo);
  }
}

// Columns of a tile's rows that no load fills, up to the next block of 64.
template <int DP>
__device__ __forceinline__ void clear_columns(float* dst, int stride, int rows, int d) {
  const int from = (d + 3) / 4 * 4, n = DP - from;
  for (int i = threadIdx.x; i < rows * n; i += SA_THREADS) dst[i / n * stride + from + i % n] = 0.f;
}

// The scores of 16 rows and 8 NT keys by a warp: s[c][e] is row g + 8 (e >> 1), key 8 c + 2 t + (e & 1), g = lane / 4, t = lane % 4.
// Which column of the head is which of a step's eight is the same for both operands, so a lane reads four columns in a row.  The tensor
// cores cut an accumulator off at each step, so large products meet there for 16 columns only, and the small ones apart (one
// accumulator for all: errors 5 times as large).
template <bool EXACT, int NT>
__device__ __forceinline__ void tile_scores(float (&s)[NT][4], const float* Qw, const float* Ks, int stride, int d) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float rest[NT][4];
#pragma unroll
  for (int c = 0; c < NT; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[c][e] = rest[c][e] = 0.f;
#pragma unroll 1
  for (int c = 0; c < d; c += 16) {
    const float4 x = *reinterpret_cast<const float4*>(Qw + g * stride + c + 4 * t), y = *reinterpret_cast<const float4*>(Qw + (g + 8) * stride + c + 4 * t);
    const Halves a0[4] = {halves<EXACT, true>(x.x), halves<EXACT, true>(y.x), halves<EXACT, true>(x.y), halves<EXACT, true>(y.y)};
    const Halves a1[4] = {halves<EXACT, true>(x.z), halves<EXACT, true>(y.z), halves<EXACT, true>(x.w), halves<EXACT, true>(y.w)};
#pragma unroll
    for (int k = 0; k < NT; k += 2) {
      Halves b0[2][2], b1[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float4 v = *reinterpret_cast<const float4*>(Ks + (8 * (k + u) + g) * stride + c + 4 * t);
        b0[u][0] = halves<EXACT, false>(v.x);
        b0[u][1] = halves<EXACT, false>(v.y);
        b1[u][0] = halves<EXACT, false>(v.z);
        b1[u][1] = halves<EXACT, false>(v.w);
      }
      float part[2][4] = {}, (&small)[2][4] = *reinterpret_cast<float(*)[2][4]>(&rest[k]);
      mma_halves<EXACT, EXACT>(part, small, a0, b0);
      mma_halves<EXACT, EXACT>(part, small, a1, b1);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[k + u][e] += part[u][e];
    }
  }
  float odd = 0.f;
#pragma unroll
  for (int c = 0; c < NT; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[c][e] += rest[c][e];
      odd = fmaf(s[c][e], 0.f, odd);
    }
  if (__builtin_expect(__any_sync(0xffffffffu, odd != 0.f), 0)) {              // what is not finite is made again from the products themselves
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int i = 0; i < d; ++i) {
        const float x = Qw[g * stride + i], y = Qw[(g + 8) * stride + i];
        const float k0 = Ks[(8 * c + 2 * t) * stride + i], k1 = Ks[(8 * c + 2 * t + 1) * stride + i];
        z[0] = fmaf(x, k0, z[0]);
        z[1] = fmaf(x, k1, z[1]);
        z[2] = fmaf(y, k0, z[2]);
        z[3] = fmaf(y, k1, z[3]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[c][e] = fabsf(s[c][e]) < INFINITY ? s[c][e] : z[e];
    }
  }
}
// in log2 units
__device__ __forceinline__ float scaled(float s, const ScoredArgs& a) {
  s *= a.scale;
  return (a.softcap > 0.f ? a.softcap * tanhf(s / a.softcap) : s) * SA_LOG2E;
}

// Floats between rows of the tiles in shared memory: 16-byte reads by 8 lanes of two rows (queries, keys) or of four rows two apart
// (values) meet no bank twice.
constexpr int qk_stride(int db) { return 64 * db + 16; }
constexpr int v_stride(int db) { return 64 * db + 4; }

// DB: blocks of 64 elements of a head.
template <typename T, int DB>
__global__ void __launch_bounds__(SA_THREADS, DB <= 2 ? 3 : 1) scored_rows_kernel(const TileArgs t) {
  extern __shared__ __align__(16) float smem[];
  constexpr int DP = 64 * DB, STRIDE = qk_stride(DB), VS = v_stride(DB);
  constexpr bool EXACT = sizeof(T) == 2;
  __shared__ long long s_q[SA_ROWS], s_at[2][ROWS_KEYS];   // where rows of q begin, and keys of this tile and the next
  float* Qs = smem;                       // [64][STRIDE]
  float* Ks = Qs + SA_ROWS * STRIDE;      // [32][STRIDE]
  float* Vs = Ks + ROWS_KEYS * STRIDE;      // [32][VS]
  pdl_prologue();
  const ScoredArgs& a = t.a;
  const int G = a.nq / a.nkv, kvh = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tt = lane & 3, d = a.d;
  // which request, which rows: the last ones, which see the most, come first
  int tile = blockIdx.x, seq = -1;
  for (int s = 0; s < a.n_seqs; ++s) {
    const int n = a.cu_q[s + 1] - a.cu_q[s];
    if (!scored_takes(a, n)) continue;
    const int nt = (n * G + SA_ROWS - 1) / SA_ROWS;
    if (tile < nt) {
      seq = s;
      tile = nt - 1 - tile;
      break;
    }
    tile -= nt;
  }
  if (seq < 0) return;
  const int first = a.cu_q[seq], n = a.cu_q[seq + 1] - first, total = min(a.kv_len[seq], a.max_keys), r0 = tile * SA_ROWS;
  const int rows = min(SA_ROWS, n * G - r0), key_begin = (int)blockIdx.z * t.p.split_tiles * ROWS_KEYS;
  const int last = min(total - n + (r0 + rows - 1) / G, total - 1);            // the newest key that a row of the tile sees
  const int all = total - n + r0 / G;                                          // every row sees keys up to here
  const int key_end = min(last + 1, key_begin + t.p.split_tiles * ROWS_KEYS);
  const T* pages = (const T*)a.pages;
  const T* values = pages + (long long)a.nkv * a.page_size * d;               // the plane behind a page's keys
  auto place = [&](int j0, long long* at) {
    if (tid < ROWS_KEYS) at[tid] = j0 + tid < key_end ? key_row(a, seq, j0 + tid, kvh, 0) : -1;
  };
  for (int r = tid; r < SA_ROWS; r += SA_THREADS)
    s_q[r] = r < rows ? (long long)(first + (r0 + r) / G) * a.q_stride + (long long)(kvh * G + (r0 + r) % G) * d : -1;
  place(key_begin, s_at[0]);
  if (d <= DP - 4) {
    clear_columns<DP>(Qs, STRIDE, SA_ROWS + ROWS_KEYS, d);
    clear_columns<DP>(Vs, VS, ROWS_KEYS, d);
  }
  __syncthreads();
  if (key_begin < key_end) {
    load_rows<T, DB, SA_ROWS>(Qs, STRIDE, (const T*)a.q, s_q, d, t.vec);
    load_rows<T, DB, ROWS_KEYS>(Ks, STRIDE, pages, s_at[0], d, t.vec);
    load_rows<T, DB, ROWS_KEYS>(Vs, VS, values, s_at[0], d, t.vec);
  }

  // rows g and g + 8 of the warp's sixteen; o[b][u][2 i + e]: row i, column 32 b + 8 tt + 4 e + u
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[2 * DB][4][4];
  int hi[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 16 * warp + g + 8 * i;
    hi[i] = r < rows ? min(total - n + (r0 + r) / G, total - 1) : -1;
  }
#pragma unroll
  for (int b = 0; b < 2 * DB; ++b)
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[b][u][e] = 0.f;
  int cur = 0;
  for (int j0 = key_begin; j0 < key_end; j0 += ROWS_KEYS, cur ^= 1) {
    const long long* at = s_at[cur];
    wait_loads<1>();                      // the keys
    // some row does not see some key of the tile
    const bool masked = __syncthreads_or(tid < ROWS_KEYS && at[tid & (ROWS_KEYS - 1)] < 0) || j0 + ROWS_KEYS - 1 > all;
    place(j0 + ROWS_KEYS, s_at[cur ^ 1]);
    float s[ROWS_KEYS / 8][4];
    tile_scores<EXACT, ROWS_KEYS / 8>(s, Qs + 16 * warp * STRIDE, Ks, STRIDE, d);
    __syncthreads();
    load_rows<T, DB, ROWS_KEYS>(Ks, STRIDE, pages, s_at[cur ^ 1], d, t.vec);       // zeros behind the last tile
    float top[2] = {-INFINITY, -INFINITY}, alpha[2];
#pragma unroll
    for (int c = 0; c < ROWS_KEYS / 8; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = 8 * c + 2 * tt + (e & 1);
        s[c][e] = scaled(s[c][e], a);
        if (masked && (j0 + j > hi[e >> 1] || at[j] < 0)) s[c][e] = -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], s[c][e]);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
      const float ref = fmaxf(m[i], top[i]), use = ref == -INFINITY ? 0.f : ref;
      alpha[i] = scored_exp2(m[i] - use);
      m[i] = ref;
      top[i] = use;
    }
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < ROWS_KEYS / 8; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[c][e] = scored_exp2(s[c][e] - top[e >> 1]);
        sum[e >> 1] += s[c][e];
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) l[i] = fmaf(l[i], alpha[i], sum[i]);           // this lane's keys; the four lanes of a row meet at the end
    wait_loads<1>();                      // the values
    __syncthreads();
#pragma unroll
    for (int b = 0; b < 2 * DB; ++b) {
      if (32 * b >= d) continue;
      // a tile's products are added up apart: an accumulator that is cut off at each step stays short
      float acc[4][4], rest[4][4];
      auto products = [&](auto all) {       // or those of the values that have halves
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[u][e] = rest[u][e] = 0.f;
#pragma unroll
        for (int c = 0; c < ROWS_KEYS / 8; ++c) {
          float4 x = *reinterpret_cast<const float4*>(Vs + (8 * c + 2 * tt) * VS + 32 * b + 4 * g);
          float4 y = *reinterpret_cast<const float4*>(Vs + (8 * c + 2 * tt + 1) * VS + 32 * b + 4 * g);
          if (!decltype(all)::value) {
            x = make_float4(fabsf(x.x) < INFINITY ? x.x : 0.f, fabsf(x.y) < INFINITY ? x.y : 0.f, fabsf(x.z) < INFINITY ? x.z : 0.f, fabsf(x.w) < INFINITY ? x.w : 0.f);
            y = make_float4(fabsf(y.x) < INFINITY ? y.x : 0.f, fabsf(y.y) < INFINITY ? y.y : 0.f, fabsf(y.z) < INFINITY ? y.z : 0.f, fabsf(y.w) < INFINITY ? y.w : 0.f);
          }
          const Halves p[4] = {halves<false, true>(s[c][0]), halves<false, true>(s[c][2]), halves<false, true>(s[c][1]), halves<false, true>(s[c][3])};
          const Halves v[4][2] = {{halves<EXACT, false>(x.x), halves<EXACT, false>(y.x)}, {halves<EXACT, false>(x.y), halves<EXACT, false>(y.y)},
                                  {halves<EXACT, false>(x.z), halves<EXACT, false>(y.z)}, {halves<EXACT, false>(x.w), halves<EXACT, false>(y.w)}};
          mma_halves<false, EXACT>(acc, rest, p, v);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[u][e] += rest[u][e];
      };
      products(std::true_type{});
      float odd = 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) odd = fmaf(acc[u][e], 0.f, odd);
      if (__builtin_expect(__any_sync(0xffffffffu, odd != 0.f), 0)) {          // a value is not finite: only who sees it multiplies by it
        products(std::false_type{});
#pragma unroll
        for (int c = 0; c < ROWS_KEYS / 8; ++c)
#pragma unroll 1
          for (int x = 0; x < 8; ++x) {
            const int j = 8 * c + x, from = (lane & ~3) | (x >> 1);
            const float even0 = __shfl_sync(0xffffffffu, s[c][0], from), odd0 = __shfl_sync(0xffffffffu, s[c][1], from);
            const float even1 = __shfl_sync(0xffffffffu, s[c][2], from), odd1 = __shfl_sync(0xffffffffu, s[c][3], from);
            const float p0 = x & 1 ? odd0 : even0, p1 = x & 1 ? odd1 : even1;
            const bool there = at[j] >= 0, sees0 = there && j0 + j <= hi[0], sees1 = there && j0 + j <= hi[1];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float v = Vs[j * VS + 32 * b + 8 * tt + 4 * e + u];
                if (fabsf(v) < INFINITY) continue;
                if (sees0) acc[u][e] = fmaf(p0, v, acc[u][e]);
                if (sees1) acc[u][2 + e] = fmaf(p1, v, acc[u][2 + e]);
              }
          }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[b][u][e] = fmaf(o[b][u][e], alpha[e >> 1], acc[u][e]);
    }
    __syncthreads();
    load_rows<T, DB, ROWS_KEYS>(Vs, VS, values, s_at[cur ^ 1], d, t.vec);
  }
  wait_loads<0>();
  T* out = (T*)a.out;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float sum = l[i];
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    const int r = 16 * warp + g + 8 * i;
    if (r >= rows) continue;
    const int token = first + (r0 + r) / G, head = kvh * G + (r0 + r) % G;
    const size_t row = (size_t)kvh * a.n_tokens * G + (size_t)first * G + r0 + r;
    const bool whole = t.p.splits == 1;
    float inv = 1.f;
    if (whole) {
      const float sink = a.sinks ? a.sinks[head] * SA_LOG2E : -INFINITY, ref = fmaxf(m[i], sink), use = ref == -INFINITY ? 0.f : ref;
      const float f = scored_exp2(m[i] - use);
      sum = fmaf(sum, f, scored_exp2(sink - use));
      inv = sum == 0.f ? 0.f : f / sum;
      if (tt == 0) a.lse[row] = sum == 0.f ? INFINITY : use + log2f(sum);
    } else if (tt == 0) {
      float* ml = t.p.ml + ((size_t)blockIdx.z * a.nkv * a.n_tokens * G + row) * 2;
      ml[0] = m[i];
      ml[1] = sum;
    }
    T* dst = out + (size_t)token * a.out_stride + (size_t)head * d;
    float* part = t.p.o + ((size_t)blockIdx.z * a.nkv * a.n_tokens * G + row) * d;
#pragma unroll
    for (int b = 0; b < 2 * DB; ++b)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int at = 32 * b + 8 * tt + 4 * e;
        if (at >= d) continue;
        float x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = o[b][u][2 * i + e] * inv;
        if (d % 4 == 0 && (!whole || (sizeof(T) == 4 && t.vec_out))) {
          *reinterpret_cast<float4*>(whole ? (float*)dst + at : part + at) = make_float4(x[0], x[1], x[2], x[3]);
          continue;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (at + u >= d) continue;
          if (whole) dst[at + u] = from_f32<T>(x[u]);
          else part[at + u] = x[u];
        }
      }
  }
}

template <typename T, int DB>
__global__ void __launch_bounds__(SA_THREADS, DB <= 2 ? 3 : 1) scored_keys_kernel(const TileArgs t) {
  extern __shared__ __align__(16) float smem[];
  constexpr int STRIDE = qk_stride(DB);
  constexpr bool EXACT = sizeof(T) == 2;
  __shared__ long long s_k[KEYS_KEYS], s_q[2][SA_ROWS];
  __shared__ float s_lse[2][SA_ROWS], s_part[SA_WARPS][KEYS_KEYS];
  float* Ks = smem;                       // [64][STRIDE]
  float* Qs = Ks + KEYS_KEYS * STRIDE;      // [64][STRIDE]
  pdl_prologue();
  const ScoredArgs& a = t.a;
  const int G = a.nq / a.nkv, kvh = blockIdx.y, seq = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tt = lane & 3, d = a.d;
  const int tiles = (int)(t.p.keys / KEYS_KEYS), chunk = blockIdx.x / tiles, key0 = (blockIdx.x - chunk * tiles) * KEYS_KEYS;
  const int first = a.cu_q[seq], n = a.cu_q[seq + 1] - first, total = min(a.kv_len[seq], a.max_keys);
  if (key0 >= total || !scored_takes(a, n)) return;
  int begin, end;
  chunk_range(t.p, n, G, total, key0, chunk, begin, end);
  if (t.p.chunks > 1 && begin >= end) return;
  auto place = [&](int i0, int buf) {
    for (int r = tid; r < SA_ROWS; r += SA_THREADS) {
      const int row = i0 * SA_ROWS + r;
      const bool in = i0 < end && row < n * G;
      s_q[buf][r] = in ? (long long)(first + row / G) * a.q_stride + (long long)(kvh * G + row % G) * d : -1;
      s_lse[buf][r] = in ? a.lse[(size_t)kvh * a.n_tokens * G + (size_t)first * G + row] : INFINITY;
    }
  };
  if (tid < KEYS_KEYS) s_k[tid] = key0 + tid < total ? key_row(a, seq, key0 + tid, kvh, 0) : -1;
  place(begin, 0);
  if (d <= 64 * DB - 4) clear_columns<64 * DB>(Ks, STRIDE, KEYS_KEYS + SA_ROWS, d);
  __syncthreads();
  if (begin < end) {
    load_rows<T, DB, KEYS_KEYS>(Ks, STRIDE, (const T*)a.pages, s_k, d, t.vec);
    load_rows<T, DB, SA_ROWS>(Qs, STRIDE, (const T*)a.q, s_q[0], d, t.vec);
  }
  float w[8][2];                          // keys 8 c + 2 tt + e
#pragma unroll
  for (int c = 0; c < 8; ++c) w[c][0] = w[c][1] = 0.f;
  int cur = 0;
  for (int i0 = begin; i0 < end; ++i0, cur ^= 1) {
    wait_loads<0>();
    __syncthreads();
    place(i0 + 1, cur ^ 1);
    float s[8][4];
    tile_scores<EXACT, KEYS_KEYS / 8>(s, Qs + 16 * warp * STRIDE, Ks, STRIDE, d);
    __syncthreads();
    load_rows<T, DB, SA_ROWS>(Qs, STRIDE, (const T*)a.q, s_q[cur ^ 1], d, t.vec);        // zeros behind the last tile
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 16 * warp + g + 8 * i, row = i0 * SA_ROWS + r, hi = row < n * G ? total - n + row / G : -1;
      const float lse = s_lse[cur][r];
#pragma unroll
      for (int c = 0; c < 8; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = scored_exp2(scaled(s[c][2 * i + e], a) - lse);
          if (key0 + 8 * c + 2 * tt + e <= hi) w[c][e] += p;
        }
    }
  }
  wait_loads<0>();
#pragma unroll
  for (int c = 0; c < 8; ++c)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) w[c][e] += __shfl_xor_sync(0xffffffffu, w[c][e], x);
      if (g == 0) s_part[warp][8 * c + 2 * tt + e] = w[c][e];
    }
  __syncthreads();
  if (tid < KEYS_KEYS && key0 + tid < total) {
    float sum = 0.f;
#pragma unroll
    for (int y = 0; y < SA_WARPS; ++y) sum += s_part[y][tid];
    if (t.p.chunks == 1) store_weight(a, seq, first, kvh, key0 + tid, key0 + tid - (total - n), sum);
    else t.p.w[(((size_t)seq * a.nkv + kvh) * t.p.chunks + chunk) * t.p.keys + key0 + tid] = sum;
  }
}

// The sums of a row's parts joined: a warp per row.
template <typename T>
__global__ void __launch_bounds__(256) scored_join_rows_kernel(const ScoredArgs a, const ScoredParts p) {
  pdl_prologue();
  const int G = a.nq / a.nkv, lane = threadIdx.x & 31;
  const size_t rows = (size_t)a.nkv * a.n_tokens * G, row = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int kvh = (int)(row / ((size_t)a.n_tokens * G)), r = (int)(row - (size_t)kvh * a.n_tokens * G), token = r / G, head = kvh * G + r % G;
  int seq = 0;                            // how many requests end at or before the token
  for (int s = 0; s < a.n_seqs; s += 32) seq += __popc(__ballot_sync(0xffffffffu, s + lane < a.n_seqs && a.cu_q[s + lane + 1] <= token));
  if (seq >= a.n_seqs) return;
  if (!scored_takes(a, a.cu_q[seq + 1] - a.cu_q[seq])) return;
  // a lane per part: its sum's reference and factor
  const float sink = a.sinks ? a.sinks[head] * SA_LOG2E : -INFINITY;
  float2 ml = make_float2(-INFINITY, 0.f);
  if (lane < p.splits) ml = *reinterpret_cast<const float2*>(p.ml + (lane * rows + row) * 2);
  float ref = fmaxf(sink, warp_max(ml.x));
  if (ref == -INFINITY) ref = 0.f;
  const float f = scored_exp2(ml.x - ref), sum = warp_sum(f * ml.y) + scored_exp2(sink - ref), inv = sum == 0.f ? 0.f : 1.0f / sum;
  T* dst = (T*)a.out + (size_t)token * a.out_stride + (size_t)head * a.d;
  if (a.d % 4 == 0) {
    for (int c0 = 0; c0 < a.d; c0 += 128) {
      const int c = c0 + 4 * lane;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int s = 0; s < p.splits; ++s) {
        const float fs = __shfl_sync(0xffffffffu, f, s);
        if (c < a.d) {
          const float4 x = *reinterpret_cast<const float4*>(p.o + (s * rows + row) * a.d + c);
          v.x = fmaf(fs, x.x, v.x); v.y = fmaf(fs, x.y, v.y); v.z = fmaf(fs, x.z, v.z); v.w = fmaf(fs, x.w, v.w);
        }
      }
      if (c < a.d) {
        dst[c] = from_f32<T>(v.x * inv);
        dst[c + 1] = from_f32<T>(v.y * inv);
        dst[c + 2] = from_f32<T>(v.z * inv);
        dst[c + 3] = from_f32<T>(v.w * inv);
      }
    }
  } else {
    for (int c0 = 0; c0 < a.d; c0 += 32) {
      const int c = c0 + lane;
      float v = 0.f;
      for (int s = 0; s < p.splits; ++s) {
        const float fs = __shfl_sync(0xffffffffu, f, s);
        if (c < a.d) v = fmaf(fs, p.o[(s * rows + row) * a.d + c], v);
      }
      if (c < a.d) dst[c] = from_f32<T>(v * inv);
    }
  }
  if (lane == 0) a.lse[row] = sum == 0.f ? INFINITY : ref + log2f(sum);
}

// The chunks' sums added in their order: a thread per key.
__global__ void __launch_bounds__(256) scored_join_keys_kernel(const ScoredArgs a, const ScoredParts p) {
  pdl_prologue();
  const int seq = blockIdx.z, kvh = blockIdx.y, key = blockIdx.x * 256 + threadIdx.x;
  const int first = a.cu_q[seq], n = a.cu_q[seq + 1] - first, total = min(a.kv_len[seq], a.max_keys);
  if (key >= total || !scored_takes(a, n)) return;
  // the chunks from the first that sees the key's tile to the last that has rows
  const int G = a.nq / a.nkv, t = key / p.tile_keys * p.tile_keys - (total - n), first_tile = t > 0 ? t * G / p.tile_rows : 0;
  const int tiles = (n * G + p.tile_rows - 1) / p.tile_rows, end = (tiles + p.chunk_tiles - 1) / p.chunk_tiles;
  const float* w = p.w + ((size_t)seq * a.nkv + kvh) * p.chunks * p.keys + key;
  float sum = 0.f;
#pragma unroll 8
  for (int c = first_tile / p.chunk_tiles; c < end; ++c) sum += w[c * p.keys];
  store_weight(a, seq, first, kvh, key, key - (total - n), sum);
}

template <typename T, int DB>
int launch_tiles(const TileArgs& t, cudaStream_t stream) {
  static std::atomic<uint64_t> rows_done{0}, keys_done{0};
  constexpr size_t rows_smem = sizeof(float) * ((SA_ROWS + ROWS_KEYS) * qk_stride(DB) + ROWS_KEYS * v_stride(DB));
  constexpr size_t keys_smem = sizeof(float) * (SA_ROWS + KEYS_KEYS) * qk_stride(DB);
  const ScoredArgs& a = t.a;
  const long long tiles = (long long)a.n_tokens * (a.nq / a.nkv) / SA_ROWS + a.n_seqs, key_tiles = (long long)(t.p.keys / KEYS_KEYS) * t.p.chunks;
  NHV_REQUIRE(tiles < (1LL << 31) && key_tiles < (1LL << 31), "scored attention: %lld tiles of rows, %lld of keys are beyond the grid's reach", tiles, key_tiles);
  NHV_CUDA(nhv_allow_smem((const void*)scored_rows_kernel<T, DB>, (int)rows_smem, rows_done), "scored attention");
  NHV_CUDA(nhv_allow_smem((const void*)scored_keys_kernel<T, DB>, (int)keys_smem, keys_done), "scored attention");
  NHV_CUDA(nhv_launch(scored_rows_kernel<T, DB>, dim3((unsigned)tiles, a.nkv, t.p.splits), SA_THREADS, rows_smem, stream, t), "scored attention");
  int rc = scored_join_rows(sizeof(T) == 4 ? NHV_F32 : NHV_BF16, a, t.p, stream);
  if (rc) return rc;
  NHV_CUDA(nhv_launch(scored_keys_kernel<T, DB>, dim3((unsigned)key_tiles, a.nkv, a.n_seqs), SA_THREADS, keys_smem, stream, t), "scored attention");
  return scored_join_keys(a, t.p, stream);
}

int tiles_at_once(int d) { return d <= 128 ? 3 * 148 : 148; }

size_t tile_parts(ScoredParts& p, int n_seqs, int n_tokens, int max_new, int max_keys, int nq, int nkv, int d) {
  p.tile_rows = SA_ROWS;
  p.tile_keys = KEYS_KEYS;
  const int at_once = tiles_at_once(d);
  return scored_parts(p, n_seqs, n_tokens, max_new, max_keys, nq, nkv, d, SA_ROWS, ROWS_KEYS, SA_ROWS * ROWS_KEYS * d / 30.0, at_once, at_once);
}

}  // namespace

size_t scored_parts(ScoredParts& p, int n_seqs, int n_tokens, int max_new, int max_keys, int nq, int nkv, int d, int row_tile, int key_tile,
                    double tile_cycles, int rows_at_once, int keys_at_once) {
  const int G = nq / nkv;
  // the rows' pass: parts of the keys where whole walks fill the SMs badly.  With `blocks` walks and `at_once` places, s parts take
  // one s-th of a walk where all run at once, else the work's share and half a part more for the last ones to end; each part's sums
  // are written and read once, 8 bytes an element at some 30 bytes a cycle.  One request's walks are alike but for the causal edge, and
  // come in whole rounds.  No part is below `least` tiles, and the sums of all parts fit 1 GiB.
  const long long blocks = ((long long)n_tokens * G / row_tile + n_seqs) * nkv;        // at most
  const int tiles = (max_keys + key_tile - 1) / key_tile, least = key_tile * row_tile >= 128 * 128 ? 8 : 3;
  const bool alike = n_seqs == 1 && max_keys >= 2 * max_new;
  int splits = 1;
  double best = 1e30;
  const double sums = row_tile * d * 8 / 30.0 / (tile_cycles * tiles);
  for (int s = 1; s <= SA_MOST_SPLITS && (s == 1 || (tiles / s >= least && s * ((size_t)n_tokens * nq * (d + 2)) <= SA_MOST_SUMS)); ++s) {
    const double waves = alike || blocks * s <= rows_at_once ? (double)((blocks * s + rows_at_once - 1) / rows_at_once) : (double)blocks * s / rows_at_once + 0.5;
    const double cost = waves / s + (s > 1 ? s * sums : 0.0);
    if (cost < best - 1e-9) {
      best = cost;
      splits = s;
    }
  }
  p.split_tiles = (tiles + splits - 1) / splits;
  p.splits = (tiles + p.split_tiles - 1) / p.split_tiles;
  // the keys' pass: chunks of rows so that two blocks come to each place that runs at once, of eight tiles at least (eight blocks and four
  // tiles: 100 against 90 us for a prompt of 2,048 tokens)
  const long long row_tiles = ((long long)max_new * G + p.tile_rows - 1) / p.tile_rows, key_tiles = (max_keys + p.tile_keys - 1) / p.tile_keys;
  const long long pairs = ((long long)n_tokens * G / p.tile_rows + n_seqs) * key_tiles * nkv;
  long long chunk = pairs / (keys_at_once * 2LL);
  if (chunk < 8) chunk = 8;
  if (chunk > row_tiles) chunk = row_tiles < 1 ? 1 : row_tiles;
  p.chunk_tiles = (int)chunk;
  p.chunks = (int)((row_tiles + chunk - 1) / chunk);
  if (p.chunks < 1) p.chunks = 1;
  p.keys = (size_t)key_tiles * p.tile_keys;
  const size_t rows = (size_t)n_tokens * nq;
  return (p.splits > 1 ? p.splits * rows * (d + 2) : 0) + (p.chunks > 1 ? (size_t)n_seqs * nkv * p.chunks * p.keys : 0) + 8;
}

// Of the rows' pass what the plan allows.  Of the keys' pass: a chunk has at least 8/9 of its share of the pairs of tiles, so a (request, KV
// head) has at most 9/8 2 keys_at_once / (key tiles x KV heads) chunks and one that is not full, of so many keys each.
size_t scored_most_parts(int n_seqs, int n_tokens, int max_keys, int nq, int nkv, int d, int tile_rows, int tile_keys, int keys_at_once) {
  const size_t sums = SA_MOST_SPLITS * ((size_t)n_tokens * nq * (d + 2)), keys = ((size_t)max_keys + tile_keys - 1) / tile_keys * tile_keys;
  const bool chunks = ((long long)n_tokens * (nq / nkv) + tile_rows - 1) / tile_rows > 8;
  return (sums < SA_MOST_SUMS ? sums : SA_MOST_SUMS) + (chunks ? n_seqs * ((size_t)keys_at_once * 9 / 4 * tile_keys + nkv * keys) : 0) + 8;
}

void scored_place(ScoredParts& p, float* work, int n_tokens, int nq, int d) {
  const size_t rows = p.splits > 1 ? (size_t)p.splits * n_tokens * nq : 0;
  p.o = work;
  p.ml = p.o + (rows * d + 3) / 4 * 4;
  p.w = p.ml + rows * 2;
}

int scored_join_rows(int dtype, const ScoredArgs& a, const ScoredParts& p, cudaStream_t stream) {
  if (p.splits <= 1 || a.n_tokens == 0) return 0;
  const dim3 grid((unsigned)(((long long)a.n_tokens * a.nq + 7) / 8));
  if (dtype == NHV_F32) NHV_CUDA(nhv_launch(scored_join_rows_kernel<float>, grid, 256, 0, stream, a, p), "scored attention");
  else NHV_CUDA(nhv_launch(scored_join_rows_kernel<__nv_bfloat16>, grid, 256, 0, stream, a, p), "scored attention");
  return 0;
}

int scored_join_keys(const ScoredArgs& a, const ScoredParts& p, cudaStream_t stream) {
  if (p.chunks <= 1) return 0;
  NHV_CUDA(nhv_launch(scored_join_keys_kernel, dim3((a.max_keys + 255) / 256, a.nkv, a.n_seqs), 256, 0, stream, a, p), "scored attention");
  return 0;
}

// What a call needs beside its arguments, and which kernels take which requests: those of up to `short_rows` rows the kernels of
// scored_attention_short.cu, the others the ones of scored_attention_tcgen05.cu, and what neither takes the kernels of this file.
struct ScoredPlan {
  bool wide;                // rows that 16-byte loads can take
  int short_rows;           // -1: none go the short way
  bool rest, many;          // there may be others; they go to the tcgen05 kernels
  ShortPlan few;
  ScoredParts parts;
  size_t floats;            // of scratch
};

static ScoredPlan scored_plan(int dtype, bool wide, int n_seqs, int n_tokens, int min_new, int max_new, int max_keys, int nq, int nkv, int d,
                              int page_size, int n_pages, int q_stride, float scale) {
  ScoredPlan p = {};
  if (n_tokens == 0) min_new = max_new = 0;       // whatever the caller's bounds say: no rows to make maps of
  p.wide = wide && d % (dtype == NHV_F32 ? 4 : 8) == 0;
  p.short_rows = -1;
  const int G = nq / nkv, most = scored_short_rows(dtype, d);
  size_t few = 0, rest = 0;
  if (p.wide && min_new <= most && scored_short_takes(dtype, min_new * G, d)) {
    p.short_rows = most;
    const int rows = max_new > most ? most : max_new * G;
    p.few = scored_short_plan(dtype, n_seqs, rows > most ? most : rows, max_keys, nkv, d);
    few = p.few.floats;
  }
  p.rest = p.short_rows < 0 || max_new > most || max_new * G > most;
  if (p.rest) {
    p.many = p.wide && scored_long_takes(dtype, nq, nkv, d, page_size, q_stride, scale);
    if (p.many) {
      rest = scored_long_plan(p.parts, n_seqs, n_tokens, max_new, max_keys, nq, nkv, d);
      p.many = scored_long_reaches(p.parts, n_seqs, n_tokens, nq, nkv, d, page_size, n_pages);
    }
    if (!p.many) rest = tile_parts(p.parts, n_seqs, n_tokens, max_new, max_keys, nq, nkv, d);
  }
  p.floats = ((size_t)n_tokens * nq + 3) / 4 * 4 + (few > rest ? few : rest);       // one after the other in the same scratch
  return p;
}

static bool scored_wide(const void* q, int q_stride, const void* out, int out_stride, const void* kv_pages) {
  return q_stride % 8 == 0 && out_stride % 8 == 0 && (uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)kv_pages % 16 == 0;
}

// A call's arguments in one block: passing them one by one costs the host more than a launch.
struct NhvScoredCall {
  const void* q;
  void* out;
  const void* kv_pages;
  const float* scores;
  float* scores_out;
  int* births;
  const int* positions;
  const int* block_table;
  const int* cu_q;
  const int* kv_len;
  const float* sinks;
  int dtype, q_stride, out_stride, bt_stride, n_seqs, n_tokens, min_new, max_new, max_kv_len, nq, nkv, d, page_size, n_pages;
  float scale, softcap;
};

static ScoredPlan scored_plan(const NhvScoredCall& c) {
  return scored_plan(c.dtype, scored_wide(c.q, c.q_stride, c.out, c.out_stride, c.kv_pages), c.n_seqs, c.n_tokens, c.min_new, c.max_new, c.max_kv_len,
                     c.nq, c.nkv, c.d, c.page_size, c.n_pages, c.q_stride, c.scale);
}

// Kilobytes of scratch that nhv_attention_scored wants for these arguments.
NHV_API int nhv_attention_scored_kilobytes(const NhvScoredCall* c) {
  if (c->n_seqs <= 0 || c->nkv <= 0 || c->nq < c->nkv || c->d <= 0 || c->page_size <= 0 || c->max_kv_len <= 0) return 0;
  return (int)(scored_plan(*c).floats * sizeof(float) / 1024 + 1);
}

// The most of any call of up to c->n_seqs requests with c->n_tokens new tokens in all and c->max_kv_len keys each.
NHV_API int nhv_attention_scored_most_kilobytes(const NhvScoredCall* c) {
  if (c->n_seqs <= 0 || c->nkv <= 0 || c->nq < c->nkv || c->d <= 0 || c->page_size <= 0 || c->max_kv_len <= 0) return 0;
  size_t most = scored_short_most(c->dtype, c->n_seqs, c->max_kv_len, c->nq / c->nkv, c->nkv, c->d);
  const size_t tiles = scored_most_parts(c->n_seqs, c->n_tokens, c->max_kv_len, c->nq, c->nkv, c->d, SA_ROWS, KEYS_KEYS, tiles_at_once(c->d));
  if (tiles > most) most = tiles;
  if (c->nq / c->nkv <= 128) {
    const size_t rows = scored_long_most(c->n_seqs, c->n_tokens, c->max_kv_len, c->nq, c->nkv, c->d);
    if (rows > most) most = rows;
  }
  return (int)((((size_t)c->n_tokens * c->nq + 3) / 4 * 4 + most) * sizeof(float) / 1024 + 1);
}

NHV_API int nhv_attention_scored(const NhvScoredCall* c, float* work, int work_kilobytes, cudaStream_t stream) {
  const int dtype = c->dtype, nq = c->nq, nkv = c->nkv, d = c->d, n_seqs = c->n_seqs, n_tokens = c->n_tokens, min_new = c->min_new, max_new = c->max_new,
            max_kv_len = c->max_kv_len;
  NHV_REQUIRE(dtype == NHV_F32 || dtype == NHV_BF16, "scored attention: unknown type %d", dtype);
  NHV_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "scored attention: %d query heads do not divide into %d KV heads", nq, nkv);
  NHV_REQUIRE(d > 0 && d <= SA_MAX_D, "scored attention: head size %d is not in 1..%d", d, SA_MAX_D);
  NHV_REQUIRE(c->page_size > 0 && c->n_pages > 0 && c->bt_stride >= 0 && nkv <= 65535, "scored attention: bad page geometry");
  NHV_REQUIRE(n_seqs >= 0 && n_tokens >= 0 && min_new >= 0 && max_new >= min_new && max_kv_len >= max_new,
              "scored attention: %d to %d new tokens with up to %d keys", min_new, max_new, max_kv_len);
  NHV_REQUIRE(c->softcap >= 0.f, "scored attention: the cap on the scores is positive");
  NHV_REQUIRE(!c->births == !c->positions || n_tokens == 0, "scored attention: births and positions go together");
  if (n_seqs == 0 || max_kv_len == 0) return 0;
  NHV_REQUIRE(n_seqs <= 65535, "scored attention: %d requests are beyond the grid's reach", n_seqs);
  ScoredPlan plan = scored_plan(*c);
  NHV_REQUIRE((size_t)work_kilobytes * 1024 >= plan.floats * sizeof(float) && (uintptr_t)work % 16 == 0, "scored attention: %d kilobytes of scratch are too few",
              work_kilobytes);
  ScoredArgs a{c->q, c->out, c->kv_pages, c->scores, c->scores_out, c->births, c->positions, c->block_table, c->cu_q, c->kv_len, c->sinks, work,
               c->q_stride, c->out_stride, c->bt_stride, n_seqs, n_tokens, nq, nkv, d, c->page_size, c->n_pages, max_kv_len, 0, 0, c->scale, c->softcap};
  float* scratch = work + ((size_t)n_tokens * nq + 3) / 4 * 4;
  // the scratch is for requests of up to max_new tokens: none takes one that brings more
  const int most_rows = max_new < 0x7fffffff / (nq / nkv) ? max_new * (nq / nkv) : 0x7fffffff;
  // The requests of many rows first: whatever can be refused is refused before anything is launched, or scores in place would hold some
  // requests' weights already.
  if (plan.rest) {
    a.min_rows = plan.short_rows + 1;
    a.max_rows = most_rows;
    scored_place(plan.parts, scratch, n_tokens, nq, d);
    int rc;
    if (plan.many) {
      rc = scored_long_launch(a, plan.parts, stream);
    } else {
      const TileArgs t{a, plan.parts, d % 4 == 0 && c->q_stride % 4 == 0 && (uintptr_t)c->q % 16 == 0 && (uintptr_t)c->kv_pages % 16 == 0,
                       c->out_stride % 4 == 0 && (uintptr_t)c->out % 16 == 0};
      const int db = d <= 64 ? 1 : d <= 128 ? 2 : 4;
      if (dtype == NHV_BF16)
        rc = db == 1 ? launch_tiles<__nv_bfloat16, 1>(t, stream) : db == 2 ? launch_tiles<__nv_bfloat16, 2>(t, stream) : launch_tiles<__nv_bfloat16, 4>(t, stream);
      else
        rc = db == 1 ? launch_tiles<float, 1>(t, stream) : db == 2 ? launch_tiles<float, 2>(t, stream) : launch_tiles<float, 4>(t, stream);
    }
    if (rc) return rc;
  }
  if (plan.short_rows < 0) return 0;
  a.min_rows = 0;
  a.max_rows = plan.short_rows < most_rows ? plan.short_rows : most_rows;
  return scored_short_launch(dtype, a, plan.few, scratch, stream);
}
