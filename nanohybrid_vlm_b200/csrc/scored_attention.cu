// Attention over cache pages that also adds up, per cached key, the weight it received: what a cache that is to drop keys
// goes by.  For every new token t of a request (n new ones, L keys in the cache with them) and query head h of KV head g
//   s[j] = cap(scale q . k[j]),  j <= L - n + t;     p[j] = exp(s[j]) / (sum_j exp(s[j]) + exp(sink[h]));     out = sum_j p[j] v[j]
//   scores_out[g][j] = (j < L - n ? scores[g][j] : 0) + sum over t and the heads of g of p[j];     births[g][j] = position, j new
// A key's sum needs the rows' final normaliser, so there are two passes: the rows' (output and log-sum), then the keys'.
//
// The entry point, and kernels for any type, size and page size that compute in fp32 on the CUDA cores (the 32-bit path, and what
// the tensor-core kernels of scored_attention_short.cu and scored_attention_tcgen05.cu refuse).
//   rows: 256 threads hold 16 RPT rows (row = token * G + head, of one request and KV head) and walk the keys in tiles of 64 through
//     shared memory.  A thread makes RPT x 4 scores from 16-byte reads along the head and RPT x 4 DB outputs, two multiply-adds
//     an instruction; P passes through shared memory.  RPT is 8 (4 for heads above 128).
//     A tile's values arrive while its scores are made, the next tile's keys while the values are used.
//   keys: 64 keys stay in shared memory, the tiles of rows pass by; a thread adds up the weights of its 4 keys, the sixteen row groups
//     meet in shared memory at the end.
// What bounds them is multiply-adds, 4 D a pair in the first and 2 D in the second, of 128 a cycle and SM, and beside them the 16-byte
// reads of shared memory, four cycles each however many lanes read the same: 12 for 128 multiply-adds a thread in the scores, 16 for
// 256 in the outputs.
// Long walks over the keys are split over blocks where there are few tiles of rows, and rows into chunks in the keys' pass; two
// small kernels join the parts in a fixed order.  No sum depends on the order in which blocks run.
//
// A key out of sight may hold anything: its score is replaced, and in tiles of which some row sees only a part its value is left
// out of that row's sum instead of being multiplied by 0.
#include "nhv_scored.cuh"

namespace {

constexpr int SA_THREADS = 256, SA_KEYS = 64;

struct TileArgs {
  ScoredArgs a;
  ScoredParts p;
  int vec;                  // rows of q and of the pages can be read four elements at a time
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

// s[i][k] = row (ty RPT + i) . key (tx + 16 k)
template <int RPT>
__device__ __forceinline__ void tile_scores(float (&s)[RPT][4], const float* Qs, const float* Ks, int stride, int d, int ty, int tx) {
  f32x2 acc[RPT][4];
#pragma unroll
  for (int i = 0; i < RPT; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[i][k] = 0ull;
  for (int c = 0; c < d; c += 4) {
    f32x2 kk[4][2];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(Ks + (tx + 16 * k) * stride + c);
      kk[k][0] = v.x;
      kk[k][1] = v.y;
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(Qs + (ty * RPT + i) * stride + c);
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[i][k] = f2_fma(q.y, kk[k][1], f2_fma(q.x, kk[k][0], acc[i][k]));
    }
  }
#pragma unroll
  for (int i = 0; i < RPT; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float x, y;
      f2_unpack(acc[i][k], x, y);
      s[i][k] = x + y;
    }
}
// in log2 units
__device__ __forceinline__ float scaled(float s, const ScoredArgs& a) {
  s *= a.scale;
  return (a.softcap > 0.f ? a.softcap * tanhf(s / a.softcap) : s) * SA_LOG2E;
}

// DB: blocks of 64 elements of a head.
template <typename T, int DB, int RPT>
__global__ void __launch_bounds__(SA_THREADS, 1) scored_rows_kernel(const TileArgs t) {
  extern __shared__ __align__(16) float smem[];
  constexpr int ROWS = 16 * RPT, DP = 64 * DB, STRIDE = DP + 4, PS = SA_KEYS + 4;
  __shared__ long long s_q[ROWS], s_at[2][SA_KEYS];      // where rows of q begin, and keys of this tile and the next
  float* Qs = smem;                       // [ROWS][STRIDE]
  float* Ks = Qs + ROWS * STRIDE;         // [64][STRIDE]
  float* Vs = Ks + SA_KEYS * STRIDE;      // [64][DP]
  float* Ps = Vs + SA_KEYS * DP;          // [ROWS][PS]
  pdl_prologue();
  const ScoredArgs& a = t.a;
  const int G = a.nq / a.nkv, kvh = blockIdx.y, tid = threadIdx.x, ty = tid >> 4, tx = tid & 15, d = a.d;
  // which request, which rows: the last ones, which see the most, come first
  int tile = blockIdx.x, seq = -1;
  for (int s = 0; s < a.n_seqs; ++s) {
    const int n = a.cu_q[s + 1] - a.cu_q[s];
    if (!scored_takes(a, n)) continue;
    const int nt = (n * G + ROWS - 1) / ROWS;
    if (tile < nt) {
      seq = s;
      tile = nt - 1 - tile;
      break;
    }
    tile -= nt;
  }
  if (seq < 0) return;
  const int first = a.cu_q[seq], n = a.cu_q[seq + 1] - first, total = min(a.kv_len[seq], a.max_keys), r0 = tile * ROWS;
  const int rows = min(ROWS, n * G - r0), key_begin = (int)blockIdx.z * t.p.split_tiles * SA_KEYS;
  const int last = min(total - n + (r0 + rows - 1) / G, total - 1);            // the newest key that a row of the tile sees
  const int all = total - n + r0 / G;                                          // every row sees keys up to here
  const int key_end = min(last + 1, key_begin + t.p.split_tiles * SA_KEYS);
  const T* pages = (const T*)a.pages;
  const T* values = pages + (long long)a.nkv * a.page_size * d;               // the plane behind a page's keys
  auto place = [&](int j0, long long* at) {
    if (tid < SA_KEYS) at[tid] = j0 + tid < key_end ? key_row(a, seq, j0 + tid, kvh, 0) : -1;
  };
  for (int r = tid; r < ROWS; r += SA_THREADS)
    s_q[r] = r < rows ? (long long)(first + (r0 + r) / G) * a.q_stride + (long long)(kvh * G + (r0 + r) % G) * d : -1;
  place(key_begin, s_at[0]);
  __syncthreads();
  if (key_begin < key_end) {
    load_rows<T, DB, ROWS>(Qs, STRIDE, (const T*)a.q, s_q, d, t.vec);
    load_rows<T, DB, SA_KEYS>(Ks, STRIDE, pages, s_at[0], d, t.vec);
    load_rows<T, DB, SA_KEYS>(Vs, DP, values, s_at[0], d, t.vec);
  }

  float m[RPT], l[RPT];
  f32x2 o[RPT][2 * DB];                   // columns 64 b + 4 tx .. + 3
  int hi[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = ty * RPT + i;
    hi[i] = r < rows ? min(total - n + (r0 + r) / G, total - 1) : -1;
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < 2 * DB; ++c) o[i][c] = 0ull;
  }
  int cur = 0;
  for (int j0 = key_begin; j0 < key_end; j0 += SA_KEYS, cur ^= 1) {
    const long long* at = s_at[cur];
    wait_loads<1>();                      // the keys
    // some row does not see some key of the tile
    const bool masked = __syncthreads_or(tid < SA_KEYS && at[tid & (SA_KEYS - 1)] < 0) || j0 + SA_KEYS - 1 > all;
    place(j0 + SA_KEYS, s_at[cur ^ 1]);
    float s[RPT][4];
    tile_scores<RPT>(s, Qs, Ks, STRIDE, d, ty, tx);
    __syncthreads();
    load_rows<T, DB, SA_KEYS>(Ks, STRIDE, pages, s_at[cur ^ 1], d, t.vec);       // zeros behind the last tile
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s[i][k] = scaled(s[i][k], a);
        if (masked && (j0 + tx + 16 * k > hi[i] || at[tx + 16 * k] < 0)) s[i][k] = -INFINITY;
        top = fmaxf(top, s[i][k]);
      }
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float ref = fmaxf(m[i], top), use = ref == -INFINITY ? 0.f : ref, alpha = scored_exp2(m[i] - use);
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s[i][k] = scored_exp2(s[i][k] - use);
        sum += s[i][k];
        Ps[(ty * RPT + i) * PS + tx + 16 * k] = s[i][k];
      }
      l[i] = fmaf(l[i], alpha, sum);      // this thread's keys; the sixteen threads of a row meet at the end
      m[i] = ref;
      const f32x2 aa = f2_pack(alpha, alpha);
#pragma unroll
      for (int c = 0; c < 2 * DB; ++c) o[i][c] = f2_mul(o[i][c], aa);
    }
    wait_loads<1>();                      // the values
    __syncthreads();
    bool each = false;
    if (masked) {                         // 0 times a value is nothing only if the value is a number
      bool odd = false;
      for (int i = tid; i < SA_KEYS * DP; i += SA_THREADS)
        if (i % DP < d) odd |= !(fabsf(Vs[i]) < INFINITY);
      each = __syncthreads_or(odd);
    }
    if (!each) {
#pragma unroll 2
      for (int j = 0; j < SA_KEYS; j += 4) {
        float4 p[RPT];
#pragma unroll
        for (int i = 0; i < RPT; ++i) p[i] = *reinterpret_cast<const float4*>(Ps + (ty * RPT + i) * PS + j);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          f32x2 v[2 * DB];
#pragma unroll
          for (int b = 0; b < DB; ++b) {
            const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(Vs + (j + k) * DP + 64 * b + 4 * tx);
            v[2 * b] = x.x;
            v[2 * b + 1] = x.y;
          }
#pragma unroll
          for (int i = 0; i < RPT; ++i) {
            const float pk = k == 0 ? p[i].x : k == 1 ? p[i].y : k == 2 ? p[i].z : p[i].w;
            const f32x2 pp = f2_pack(pk, pk);
#pragma unroll
            for (int c = 0; c < 2 * DB; ++c) o[i][c] = f2_fma(pp, v[c], o[i][c]);
          }
        }
      }
    } else {
      for (int j = 0; j < SA_KEYS && j0 + j < key_end; ++j) {
        if (at[j] < 0) continue;
        f32x2 v[2 * DB];
#pragma unroll
        for (int b = 0; b < DB; ++b) {
          const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(Vs + j * DP + 64 * b + 4 * tx);
          v[2 * b] = x.x;
          v[2 * b + 1] = x.y;
        }
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          if (j0 + j > hi[i]) continue;
          const float pk = Ps[(ty * RPT + i) * PS + j];
          const f32x2 pp = f2_pack(pk, pk);
#pragma unroll
          for (int c = 0; c < 2 * DB; ++c) o[i][c] = f2_fma(pp, v[c], o[i][c]);
        }
      }
    }
    __syncthreads();
    load_rows<T, DB, SA_KEYS>(Vs, DP, values, s_at[cur ^ 1], d, t.vec);
  }
  wait_loads<0>();
  T* out = (T*)a.out;
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    float sum = l[i];
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    const int r = ty * RPT + i;
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
      if (tx == 0) a.lse[row] = sum == 0.f ? INFINITY : use + log2f(sum);
    } else if (tx == 0) {
      float* ml = t.p.ml + ((size_t)blockIdx.z * a.nkv * a.n_tokens * G + row) * 2;
      ml[0] = m[i];
      ml[1] = sum;
    }
#pragma unroll
    for (int c = 0; c < 2 * DB; ++c) {
      float x, y;
      f2_unpack(o[i][c], x, y);
      const int at = 64 * (c >> 1) + 4 * tx + 2 * (c & 1);
      if (whole) {
        T* dst = out + (size_t)token * a.out_stride + (size_t)head * d + at;
        if (at < d) dst[0] = from_f32<T>(x * inv);
        if (at + 1 < d) dst[1] = from_f32<T>(y * inv);
      } else {
        float* dst = t.p.o + ((size_t)blockIdx.z * a.nkv * a.n_tokens * G + row) * d + at;
        if (at < d) dst[0] = x;
        if (at + 1 < d) dst[1] = y;
      }
    }
  }
}

template <typename T, int DB, int RPT>
__global__ void __launch_bounds__(SA_THREADS, 1) scored_keys_kernel(const TileArgs t) {
  extern __shared__ __align__(16) float smem[];
  constexpr int ROWS = 16 * RPT, STRIDE = 64 * DB + 4;
  __shared__ long long s_k[SA_KEYS], s_q[2][ROWS];
  __shared__ float s_lse[2][ROWS], s_part[16][SA_KEYS];
  float* Ks = smem;                       // [64][STRIDE]
  float* Qs = Ks + SA_KEYS * STRIDE;      // [2][ROWS][STRIDE]
  pdl_prologue();
  const ScoredArgs& a = t.a;
  const int G = a.nq / a.nkv, kvh = blockIdx.y, seq = blockIdx.z, tid = threadIdx.x, ty = tid >> 4, tx = tid & 15, d = a.d;
  const int tiles = (int)(t.p.keys / SA_KEYS), chunk = blockIdx.x / tiles, key0 = (blockIdx.x - chunk * tiles) * SA_KEYS;
  const int first = a.cu_q[seq], n = a.cu_q[seq + 1] - first, total = min(a.kv_len[seq], a.max_keys);
  if (key0 >= total || !scored_takes(a, n)) return;
  int begin, end;
  chunk_range(t.p, n, G, total, key0, chunk, begin, end);
  if (t.p.chunks > 1 && begin >= end) return;
  auto place = [&](int i0, int buf) {
    for (int r = tid; r < ROWS; r += SA_THREADS) {
      const int row = i0 * ROWS + r;
      const bool in = i0 < end && row < n * G;
      s_q[buf][r] = in ? (long long)(first + row / G) * a.q_stride + (long long)(kvh * G + row % G) * d : -1;
      s_lse[buf][r] = in ? a.lse[(size_t)kvh * a.n_tokens * G + (size_t)first * G + row] : INFINITY;
    }
  };
  if (tid < SA_KEYS) s_k[tid] = key0 + tid < total ? key_row(a, seq, key0 + tid, kvh, 0) : -1;
  place(begin, 0);
  __syncthreads();
  if (begin < end) {
    load_rows<T, DB, SA_KEYS>(Ks, STRIDE, (const T*)a.pages, s_k, d, t.vec);
    load_rows<T, DB, ROWS>(Qs, STRIDE, (const T*)a.q, s_q[0], d, t.vec);
  }
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  int cur = 0;
  for (int i0 = begin; i0 < end; ++i0, cur ^= 1) {
    place(i0 + 1, cur ^ 1);
    __syncthreads();
    load_rows<T, DB, ROWS>(Qs + (cur ^ 1) * ROWS * STRIDE, STRIDE, (const T*)a.q, s_q[cur ^ 1], d, t.vec);      // zeros behind the last tile
    wait_loads<1>();
    __syncthreads();
    float s[RPT][4];
    tile_scores<RPT>(s, Qs + cur * ROWS * STRIDE, Ks, STRIDE, d, ty, tx);
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int r = ty * RPT + i, row = i0 * ROWS + r, hi = row < n * G ? total - n + row / G : -1;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float p = scored_exp2(scaled(s[i][k], a) - s_lse[cur][r]);
        if (key0 + tx + 16 * k <= hi) w[k] += p;
      }
    }
    __syncthreads();
  }
  wait_loads<0>();
#pragma unroll
  for (int k = 0; k < 4; ++k) s_part[ty][tx + 16 * k] = w[k];
  __syncthreads();
  if (tid < SA_KEYS && key0 + tid < total) {
    float sum = 0.f;
#pragma unroll
    for (int y = 0; y < 16; ++y) sum += s_part[y][tid];
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

template <typename T, int DB, int RPT>
int launch_tiles(const TileArgs& t, cudaStream_t stream) {
  static std::atomic<uint64_t> rows_done{0}, keys_done{0};
  constexpr int ROWS = 16 * RPT, STRIDE = 64 * DB + 4;
  constexpr size_t rows_smem = sizeof(float) * ((ROWS + SA_KEYS) * STRIDE + SA_KEYS * 64 * DB + ROWS * (SA_KEYS + 4));
  constexpr size_t keys_smem = sizeof(float) * (2 * ROWS + SA_KEYS) * STRIDE;
  const ScoredArgs& a = t.a;
  const long long tiles = (long long)a.n_tokens * (a.nq / a.nkv) / ROWS + a.n_seqs, key_tiles = (long long)(t.p.keys / SA_KEYS) * t.p.chunks;
  NHV_REQUIRE(tiles < (1LL << 31) && key_tiles < (1LL << 31), "scored attention: %lld tiles of rows, %lld of keys are beyond the grid's reach", tiles, key_tiles);
  NHV_CUDA(nhv_allow_smem((const void*)scored_rows_kernel<T, DB, RPT>, (int)rows_smem, rows_done), "scored attention");
  NHV_CUDA(nhv_allow_smem((const void*)scored_keys_kernel<T, DB, RPT>, (int)keys_smem, keys_done), "scored attention");
  NHV_CUDA(nhv_launch(scored_rows_kernel<T, DB, RPT>, dim3((unsigned)tiles, a.nkv, t.p.splits), SA_THREADS, rows_smem, stream, t), "scored attention");
  int rc = scored_join_rows(sizeof(T) == 4 ? NHV_F32 : NHV_BF16, a, t.p, stream);
  if (rc) return rc;
  NHV_CUDA(nhv_launch(scored_keys_kernel<T, DB, RPT>, dim3((unsigned)key_tiles, a.nkv, a.n_seqs), SA_THREADS, keys_smem, stream, t), "scored attention");
  return scored_join_keys(a, t.p, stream);
}

// Rows of a thread of the tiles' sixteen row groups.
int rows_per_thread(int d) { return d <= 128 ? 8 : 4; }

size_t tile_parts(ScoredParts& p, int n_seqs, int n_tokens, int max_new, int max_keys, int nq, int nkv, int d) {
  p.tile_rows = 16 * rows_per_thread(d);
  p.tile_keys = SA_KEYS;
  return scored_parts(p, n_seqs, n_tokens, max_new, max_keys, nq, nkv, d, p.tile_rows, SA_KEYS, p.tile_rows * SA_KEYS * d / 50.0, 148, 148);
}

}  // namespace

size_t scored_parts(ScoredParts& p, int n_seqs, int n_tokens, int max_new, int max_keys, int nq, int nkv, int d, int row_tile, int key_tile,
                    double tile_cycles, int rows_at_once, int keys_at_once) {
  const int G = nq / nkv;
  // the rows' pass: parts of the keys where whole walks fill the SMs badly.  With `blocks` walks and `at_once` places, s parts take
  // one s-th of a walk where all run at once, else the work's share and half a part more for the last ones to end; each part's sums
  // are written and read once, 8 bytes an element at some 30 bytes a cycle.  One request's walks are alike but for the causal edge, and
  // come in whole rounds.  No part is below `least` tiles.
  const long long blocks = ((long long)n_tokens * G / row_tile + n_seqs) * nkv;        // at most
  const int tiles = (max_keys + key_tile - 1) / key_tile, least = key_tile * row_tile >= 128 * 128 ? 8 : 3;
  const bool alike = n_seqs == 1 && max_keys >= 2 * max_new;
  int splits = 1;
  double best = 1e30;
  const double sums = row_tile * d * 8 / 30.0 / (tile_cycles * tiles);
  for (int s = 1; s <= 32 && (s == 1 || tiles / s >= least); ++s) {
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

void scored_place(ScoredParts& p, float* work, int n_tokens, int nq, int d) {
  const size_t rows = p.splits > 1 ? (size_t)p.splits * n_tokens * nq : 0;
  p.o = work;
  p.ml = p.o + (rows * d + 3) / 4 * 4;
  p.w = p.ml + rows * 2;
}

int scored_join_rows(int dtype, const ScoredArgs& a, const ScoredParts& p, cudaStream_t stream) {
  if (p.splits <= 1) return 0;
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
                              int page_size, float scale) {
  ScoredPlan p = {};
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
    p.many = p.wide && scored_long_takes(dtype, nq, nkv, d, page_size, scale);
    rest = p.many ? scored_long_plan(p.parts, n_seqs, n_tokens, max_new, max_keys, nq, nkv, d)
                  : tile_parts(p.parts, n_seqs, n_tokens, max_new, max_keys, nq, nkv, d);
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
                     c.nq, c.nkv, c.d, c.page_size, c.scale);
}

// Kilobytes of scratch that nhv_attention_scored wants for these arguments.
NHV_API int nhv_attention_scored_kilobytes(const NhvScoredCall* c) {
  if (c->n_seqs <= 0 || c->nkv <= 0 || c->nq < c->nkv || c->d <= 0 || c->page_size <= 0 || c->max_kv_len <= 0) return 0;
  return (int)(scored_plan(*c).floats * sizeof(float) / 1024 + 1);
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
               c->q_stride, c->out_stride, c->bt_stride, n_seqs, n_tokens, nq, nkv, d, c->page_size, c->n_pages, max_kv_len, 0, 0x7fffffff, c->scale, c->softcap};
  float* scratch = work + ((size_t)n_tokens * nq + 3) / 4 * 4;
  if (plan.short_rows >= 0) {
    a.max_rows = plan.short_rows;
    const int rc = scored_short_launch(dtype, a, plan.few, scratch, stream);
    if (rc || !plan.rest) return rc;
    a.min_rows = plan.short_rows + 1;
    a.max_rows = 0x7fffffff;
  }
  scored_place(plan.parts, scratch, n_tokens, nq, d);
  if (plan.many) return scored_long_launch(a, plan.parts, stream);
  const TileArgs t{a, plan.parts, d % 4 == 0 && c->q_stride % 4 == 0 && (uintptr_t)c->q % 16 == 0 && (uintptr_t)c->kv_pages % 16 == 0};
  const int db = d <= 64 ? 1 : d <= 128 ? 2 : 4;
  if (dtype == NHV_BF16)
    return db == 1 ? launch_tiles<__nv_bfloat16, 1, 8>(t, stream) : db == 2 ? launch_tiles<__nv_bfloat16, 2, 8>(t, stream) : launch_tiles<__nv_bfloat16, 4, 4>(t, stream);
  return db == 1 ? launch_tiles<float, 1, 8>(t, stream) : db == 2 ? launch_tiles<float, 2, 8>(t, stream) : launch_tiles<float, 4, 4>(t, stream);
}
