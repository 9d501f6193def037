// Attention over cache pages that also adds up, per cached key, the weight it received: what a cache that is to drop keys
// goes by.  For every new token t of a request (n new ones, L keys in the cache with them) and query head h of KV head g
//   s[j] = cap(scale q . k[j]),  j <= L - n + t;     p[j] = exp(s[j]) / (sum_j exp(s[j]) + exp(sink[h]));     out = sum_j p[j] v[j]
//   scores_out[g][j] = (j < L - n ? scores[g][j] : 0) + sum over t and the heads of g of p[j];     births[g][j] = position, j new
// A key's sum needs the rows' final normaliser, so there are two passes: the rows' (output and log-sum), then the keys'.
//
// The kernels of this file take any type, size and page size and compute in fp32.
//   rows: a block holds 16 rows (token, head) of a KV head; 32 keys at a time in shared memory, lane <-> key for the scores,
//     lane <-> column for the output.
//   keys: a block holds 32 keys of a request and KV head and walks the rows that see them, lane <-> key, the warps' sums added
//     in a fixed order at the end.
// No sum is shared between blocks, so results do not depend on the order in which blocks run.
#include "nhv_scored.cuh"

namespace {

constexpr int SA_WARPS = 4, SA_ROWS_PER_WARP = 4, SA_ROWS = SA_WARPS * SA_ROWS_PER_WARP, SA_KEYS = 32;

__device__ __forceinline__ float capped(float s, float cap) { return cap > 0.f ? cap * tanhf(s / cap) : s; }

template <typename T>
__global__ void __launch_bounds__(SA_WARPS * 32) scored_rows_kernel(const ScoredArgs a) {
  extern __shared__ float smem[];
  __shared__ long long k_at[SA_KEYS], v_at[SA_KEYS];
  pdl_prologue();
  const int G = a.nq / a.nkv, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // a tile is a whole number of tokens where a group fits the 16 rows, else 16 heads of one token
  const int per_tile = SA_ROWS / G > 0 ? SA_ROWS / G : 1, head_blocks = (G + SA_ROWS - 1) / SA_ROWS;
  int tile = blockIdx.x / head_blocks;
  const int g0 = (blockIdx.x % head_blocks) * SA_ROWS, gs = min(G - g0, SA_ROWS);
  const int seq = find_tile(a, per_tile, tile);
  if (seq < 0) return;
  const int first = a.cu_q[seq], n = a.cu_q[seq + 1] - first, total = min(a.kv_len[seq], a.max_keys), t0 = tile * per_tile;
  const int rows = min(per_tile, n - t0) * gs, d = a.d, ks = d + 1;
  float* Qs = smem;                       // [16][d]
  float* Ks = Qs + SA_ROWS * d;           // [32][d + 1]
  float* Vs = Ks + SA_KEYS * ks;          // [32][d]
  float* Ps = Vs + SA_KEYS * d;           // [warps][32]
  const T* q = (const T*)a.q;
  const T* pages = (const T*)a.pages;
  for (int i = threadIdx.x; i < rows * d; i += blockDim.x) {
    const int r = i / d, c = i - r * d;
    Qs[i] = to_f32<T>(q[(size_t)(first + t0 + r / gs) * a.q_stride + (size_t)(kvh * G + g0 + r % gs) * d + c]);
  }
  float m[SA_ROWS_PER_WARP], l[SA_ROWS_PER_WARP], o[SA_ROWS_PER_WARP][SA_MAX_D / 32];
#pragma unroll
  for (int i = 0; i < SA_ROWS_PER_WARP; ++i) {
    const int r = warp * SA_ROWS_PER_WARP + i;
    const bool sink = a.sinks && r < rows;
    m[i] = sink ? a.sinks[kvh * G + g0 + r % gs] : -INFINITY;
    l[i] = sink ? 1.f : 0.f;
#pragma unroll
    for (int c = 0; c < SA_MAX_D / 32; ++c) o[i][c] = 0.f;
  }
  const int last = min(total - n + t0 + (rows - 1) / gs, total - 1);       // the newest key that a row of the tile sees
  for (int j0 = 0; j0 <= last; j0 += SA_KEYS) {
    __syncthreads();
    if (threadIdx.x < SA_KEYS) {
      const int j = j0 + threadIdx.x;
      k_at[threadIdx.x] = j <= last ? key_row(a, seq, j, kvh, 0) : -1;
      v_at[threadIdx.x] = j <= last ? key_row(a, seq, j, kvh, 1) : -1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < SA_KEYS * d; i += blockDim.x) {
      const int r = i / d, c = i - r * d;
      Ks[r * ks + c] = k_at[r] >= 0 ? to_f32<T>(pages[k_at[r] + c]) : 0.f;
      Vs[i] = v_at[r] >= 0 ? to_f32<T>(pages[v_at[r] + c]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SA_ROWS_PER_WARP; ++i) {
      const int r = warp * SA_ROWS_PER_WARP + i;
      if (r >= rows) break;
      const int hi = total - n + t0 + r / gs;
      const bool sees = j0 + lane <= hi && k_at[lane] >= 0;
      float s = 0.f;
      for (int c = 0; c < d; ++c) s = fmaf(Qs[r * d + c], Ks[lane * ks + c], s);
      s = sees ? capped(s * a.scale, a.softcap) : -INFINITY;
      const float top = warp_max(s);
      const unsigned live = __ballot_sync(0xffffffffu, sees);
      if (!live) continue;
      const float m_new = fmaxf(m[i], top), ref = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = expf(m[i] - ref), p = sees ? expf(s - ref) : 0.f;
      l[i] = l[i] * alpha + warp_sum(p);
      m[i] = m_new;
      Ps[warp * SA_KEYS + lane] = p;
      __syncwarp();
#pragma unroll
      for (int c = 0; c < SA_MAX_D / 32; ++c) {
        if (c * 32 + lane < d) {
          float acc = 0.f;
          for (int k = 0; k < SA_KEYS; ++k)
            if (live >> k & 1) acc = fmaf(Ps[warp * SA_KEYS + k], Vs[k * d + c * 32 + lane], acc);   // a key out of sight may hold anything
          o[i][c] = o[i][c] * alpha + acc;
        }
      }
      __syncwarp();
    }
  }
  T* out = (T*)a.out;
#pragma unroll
  for (int i = 0; i < SA_ROWS_PER_WARP; ++i) {
    const int r = warp * SA_ROWS_PER_WARP + i;
    if (r >= rows) break;
    const int token = first + t0 + r / gs, head = g0 + r % gs;
    const float inv = l[i] == 0.f ? 0.f : 1.0f / l[i];
#pragma unroll
    for (int c = 0; c < SA_MAX_D / 32; ++c)
      if (c * 32 + lane < d) out[(size_t)token * a.out_stride + (size_t)(kvh * G + head) * d + c * 32 + lane] = from_f32<T>(o[i][c] * inv);
    if (lane == 0) a.lse[((size_t)kvh * a.n_tokens + token) * G + head] = l[i] == 0.f ? INFINITY : fmaf(m[i], SA_LOG2E, log2f(l[i]));
  }
}

template <typename T>
__global__ void __launch_bounds__(SA_WARPS * 32) scored_keys_kernel(const ScoredArgs a) {
  extern __shared__ float smem[];
  __shared__ float part[SA_WARPS][SA_KEYS];
  pdl_prologue();
  const int G = a.nq / a.nkv, kvh = blockIdx.y, seq = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = a.cu_q[seq], n = a.cu_q[seq + 1] - first, total = min(a.kv_len[seq], a.max_keys), j0 = blockIdx.x * SA_KEYS;
  if (j0 >= total || !scored_takes(a, n)) return;
  const int d = a.d, ks = d + 1, j = j0 + lane;
  float* Ks = smem;                       // [32][d + 1]
  float* Qs = Ks + SA_KEYS * ks;          // [warps][d]
  const T* q = (const T*)a.q;
  const T* pages = (const T*)a.pages;
  for (int i = threadIdx.x; i < SA_KEYS * d; i += blockDim.x) {
    const int r = i / d, c = i - r * d;
    const long long at = j0 + r < total ? key_row(a, seq, j0 + r, kvh, 0) : -1;
    Ks[r * ks + c] = at >= 0 ? to_f32<T>(pages[at + c]) : 0.f;
  }
  __syncthreads();
  const int t_first = max(0, j0 - (total - n));        // the first token that sees a key of the block
  float w = 0.f;
  for (int r = t_first * G + warp; r < n * G; r += SA_WARPS) {
    const int t = r / G, h = r - t * G;
    __syncwarp();
    for (int c = lane; c < d; c += 32) Qs[warp * d + c] = to_f32<T>(q[(size_t)(first + t) * a.q_stride + (size_t)(kvh * G + h) * d + c]);
    __syncwarp();
    float s = 0.f;
    for (int c = 0; c < d; ++c) s = fmaf(Qs[warp * d + c], Ks[lane * ks + c], s);
    if (j <= total - n + t)
      w += exp2f(fmaf(capped(s * a.scale, a.softcap), SA_LOG2E, -a.lse[((size_t)kvh * a.n_tokens + first + t) * G + h]));
  }
  part[warp][lane] = w;
  __syncthreads();
  if (warp == 0 && j < total) {
    float sum = part[0][lane];
    for (int k = 1; k < SA_WARPS; ++k) sum += part[k][lane];
    store_weight(a, seq, first, kvh, j, j - (total - n), sum);
  }
}

template <typename T>
int launch_simt(const ScoredArgs& a, int max_kv_len, cudaStream_t stream) {
  static std::atomic<uint64_t> rows_done{0}, keys_done{0};
  const int G = a.nq / a.nkv, per_tile = SA_ROWS / G > 0 ? SA_ROWS / G : 1, head_blocks = (G + SA_ROWS - 1) / SA_ROWS;
  const size_t rows_smem = sizeof(float) * (SA_ROWS * a.d + SA_KEYS * (a.d + 1) + SA_KEYS * a.d + SA_WARPS * SA_KEYS);
  const size_t keys_smem = sizeof(float) * (SA_KEYS * (a.d + 1) + SA_WARPS * a.d);
  const long long tiles = ((long long)a.n_tokens / per_tile + a.n_seqs) * head_blocks;
  NHV_REQUIRE(tiles < (1LL << 31), "scored attention: %lld tiles of new tokens are beyond the grid's reach", tiles);
  NHV_CUDA(nhv_allow_smem((const void*)scored_rows_kernel<T>, 96 * 1024, rows_done), "scored attention");
  NHV_CUDA(nhv_allow_smem((const void*)scored_keys_kernel<T>, 96 * 1024, keys_done), "scored attention");
  NHV_CUDA(nhv_launch(scored_rows_kernel<T>, dim3((unsigned)tiles, a.nkv), SA_WARPS * 32, rows_smem, stream, a), "scored attention");
  NHV_CUDA(nhv_launch(scored_keys_kernel<T>, dim3((max_kv_len + SA_KEYS - 1) / SA_KEYS, a.nkv, a.n_seqs), SA_WARPS * 32, keys_smem, stream, a),
           "scored attention");
  return 0;
}

}  // namespace

// What a call needs beside its arguments, and which kernels take which requests: those of up to `short_rows` rows the kernels of
// scored_attention_short.cu, the others the ones of scored_attention_tcgen05.cu, and what neither takes the kernels of this file.
struct ScoredPlan {
  int short_rows;           // -1: none go that way
  bool many;                // requests above that go to the tcgen05 kernels
  ShortPlan few;
  LongPlan rest;
  size_t floats;            // of scratch
};

static ScoredPlan scored_plan(int dtype, int n_seqs, int n_tokens, int min_new, int max_new, int max_keys, int nq, int nkv, int d, int page_size,
                              float scale) {
  ScoredPlan p = {};
  p.short_rows = -1;
  const int G = nq / nkv, most = d <= 128 ? 16 : 8;
  size_t floats = 0;
  if (scored_short_takes(dtype, min_new * G, d)) {
    p.short_rows = most;
    const int rows = max_new > most ? most : max_new * G;
    p.few = scored_short_plan(dtype, n_seqs, rows > most ? most : rows, max_keys, nkv, d);
    floats = p.few.floats;
  }
  p.many = max_new > most || max_new * G > p.short_rows;
  if (p.many) p.many = scored_long_takes(dtype, nq, nkv, d, page_size, scale);
  if (p.many) {
    p.rest = scored_long_plan(n_seqs, n_tokens, max_new, max_keys, nq, nkv, d);
    if (p.rest.floats > floats) floats = p.rest.floats;      // one after the other in the same scratch
  }
  p.floats = ((size_t)n_tokens * nq + 3) / 4 * 4 + floats;
  return p;
}

// Kilobytes of scratch that nhv_attention_scored wants for a call of these sizes.
NHV_API int nhv_attention_scored_kilobytes(int dtype, int n_seqs, int n_tokens, int min_new, int max_new, int max_kv_len, int nq, int nkv, int d,
                                           int page_size, float scale) {
  if (n_seqs <= 0 || nkv <= 0 || nq < nkv || d <= 0 || page_size <= 0) return 0;
  return (int)(scored_plan(dtype, n_seqs, n_tokens, min_new, max_new, max_kv_len, nq, nkv, d, page_size, scale).floats * sizeof(float) / 1024 + 1);
}

NHV_API int nhv_attention_scored(int dtype, const void* q, int q_stride, void* out, int out_stride, const void* kv_pages,
                                 const float* scores, float* scores_out, int* births, const int* positions, const int* block_table,
                                 int bt_stride, const int* cu_q, const int* kv_len, int n_seqs, int n_tokens, int min_new, int max_new,
                                 int max_kv_len, int nq, int nkv, int d, int page_size, int n_pages, float scale, const float* sinks,
                                 float softcap, float* work, int work_kilobytes, cudaStream_t stream) {
  NHV_REQUIRE(dtype == NHV_F32 || dtype == NHV_BF16, "scored attention: unknown type %d", dtype);
  NHV_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "scored attention: %d query heads do not divide into %d KV heads", nq, nkv);
  NHV_REQUIRE(d > 0 && d <= SA_MAX_D, "scored attention: head size %d is not in 1..%d", d, SA_MAX_D);
  NHV_REQUIRE(page_size > 0 && n_pages > 0 && bt_stride >= 0 && nkv <= 65535, "scored attention: bad page geometry");
  NHV_REQUIRE(n_seqs >= 0 && n_tokens >= 0 && min_new >= 0 && max_new >= min_new && max_kv_len >= max_new,
              "scored attention: %d to %d new tokens with up to %d keys", min_new, max_new, max_kv_len);
  NHV_REQUIRE(softcap >= 0.f, "scored attention: the cap on the scores is positive");
  NHV_REQUIRE(!births == !positions || n_tokens == 0, "scored attention: births and positions go together");
  if (n_seqs == 0 || max_kv_len == 0) return 0;
  NHV_REQUIRE(n_seqs <= 65535, "scored attention: %d requests are beyond the grid's reach", n_seqs);
  // rows that 16-byte loads cannot take go to the kernels of this file
  const bool wide = d % 8 == 0 && q_stride % 8 == 0 && out_stride % 8 == 0 && (uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 &&
                    (uintptr_t)kv_pages % 16 == 0;
  const ScoredPlan plan = scored_plan(dtype, n_seqs, n_tokens, min_new, max_new, max_kv_len, nq, nkv, d, page_size, scale);
  NHV_REQUIRE((size_t)work_kilobytes * 1024 >= plan.floats * sizeof(float) && (uintptr_t)work % 16 == 0, "scored attention: %d kilobytes of scratch are too few",
              work_kilobytes);
  ScoredArgs a{q, out, kv_pages, scores, scores_out, births, positions, block_table, cu_q, kv_len, sinks, work,
               q_stride, out_stride, bt_stride, n_seqs, n_tokens, nq, nkv, d, page_size, n_pages, max_kv_len, 0, 0x7fffffff, scale, softcap};
  float* scratch = work + ((size_t)n_tokens * nq + 3) / 4 * 4;
  if (wide && plan.short_rows >= 0) {
    a.max_rows = plan.short_rows;
    const int rc = scored_short_launch(dtype, a, plan.few, scratch, stream);
    if (rc) return rc;
    if (max_new <= plan.short_rows && max_new * (nq / nkv) <= plan.short_rows) return 0;
    a.min_rows = plan.short_rows + 1;
    a.max_rows = 0x7fffffff;
  }
  if (wide && plan.many) return scored_long_launch(a, plan.rest, scratch, stream);
  return dtype == NHV_F32 ? launch_simt<float>(a, max_kv_len, stream) : launch_simt<__nv_bfloat16>(a, max_kv_len, stream);
}
