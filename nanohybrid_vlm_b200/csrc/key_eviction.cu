// Dropping keys from a paged cache by the attention weight that they have gathered (their scores).
//
// The choice, per request and KV head.  The keys of the first `keep_first` positions and of the last `keep_recent` count as
// +inf, a score that is no number as less than any; the `budget` largest stay, of equal ones those in the lowest slots.  It is said
// as moves: the i-th kept slot at or above the budget is the source for the i-th dropped slot below it.  After the moves the request's
// keys fill the slots [0, budget), in no order, which attention does not need; births say which position a slot holds.
// Every source lies at or above the budget and every target below it, so the moves may run in any order, and may run twice.
//
//   choice: a block per (request, KV head).  The bound is the budget-th largest of the scores as whole numbers of the same
//     order, found eight bits at a time from counts in shared memory; the last pass goes over the slots in order and numbers
//     sources and targets by prefix sums over the block.  Reads 8 bytes a key, four times at most (L2 after the first).
//   moves: a warp per move carries the K row, the V row, the score and the birth.
#include "nhv_common.cuh"

namespace {

constexpr int EV_THREADS = 512;

__device__ int g_key_eviction_error = 0;      // 1: a request had more moves than the caller made room for

// A score as a whole number of the same order: -0 as 0, no number below everything.
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct ChoiceArgs {
  const float* scores;
  const int* births;
  const int* block_table;
  const int* kv_len;
  const int* seen;          // per request: the position that comes next
  const int* budgets;
  int* sources;             // [n_seqs, nkv, max_moves], -1 behind a request's last move
  int* targets;
  int bt_stride, nkv, page_size, n_pages, max_moves, keep_first, keep_recent;
  int max_keys;             // what the caller says of kv_len: no table is read beyond it
};

__device__ __forceinline__ uint32_t key_of(const ChoiceArgs& a, int seq, int kvh, int j, int recent) {
  const int page = a.block_table[(size_t)seq * a.bt_stride + j / a.page_size];
  if (page < 0 || page >= a.n_pages) return 0u;
  const size_t at = ((size_t)page * a.nkv + kvh) * a.page_size + j % a.page_size;
  const int birth = a.births[at];
  return birth < a.keep_first || birth >= recent ? ordered(INFINITY) : ordered(a.scores[at]);
}

// Exclusive prefix sums of two counts packed in one word, over the block.
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t* red, uint32_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (int w = 0; w < EV_THREADS / 32; ++w) {
    if (w < warp) before += red[w];
    all += red[w];
  }
  total = all;
  return before + x - v;
}

__global__ void __launch_bounds__(EV_THREADS) select_keys_kernel(const ChoiceArgs a) {
  __shared__ int count[256];
  __shared__ uint32_t red[EV_THREADS / 32];
  __shared__ uint32_t s_bound;
  __shared__ int s_need;
  pdl_prologue();
  const int kvh = blockIdx.x, seq = blockIdx.y, L = min(a.kv_len[seq], a.max_keys), budget = max(0, a.budgets[seq]);
  const int recent = a.seen[seq] - a.keep_recent;
  int* sources = a.sources + ((size_t)seq * a.nkv + kvh) * a.max_moves;
  int* targets = a.targets + ((size_t)seq * a.nkv + kvh) * a.max_moves;
  int moves = 0;
  if (L > budget) {
    uint32_t bound = 0, mask = 0;
    int need = budget;                                  // how many of the keys that agree with `bound` so far are kept
    for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
      for (int i = threadIdx.x; i < 256; i += EV_THREADS) count[i] = 0;
      __syncthreads();
      for (int j = threadIdx.x; j < L; j += EV_THREADS) {
        const uint32_t k = key_of(a, seq, kvh, j, recent);
        if ((k & mask) == bound) atomicAdd(&count[k >> shift & 255], 1);
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        int above = 0, digit = 255;
        while (above + count[digit] < need) above += count[digit--];
        s_bound = bound | (uint32_t)digit << shift;
        s_need = need - above;
      }
      __syncthreads();
      bound = s_bound;
      need = s_need;
      mask |= 255u << shift;
    }
    // keys above the bound stay, and the first `need` of those equal to it
    int equal_before = 0, source_before = 0, target_before = 0;
    for (int j0 = 0; j0 < L; j0 += EV_THREADS) {
      const int j = j0 + threadIdx.x;
      const uint32_t k = j < L ? key_of(a, seq, kvh, j, recent) : 0u;
      const bool equal = j < L && need > 0 && k == bound;
      uint32_t all;
      const uint32_t e = block_prefix(equal ? 1u : 0u, red, all);
      const bool kept = j < L && budget > 0 && (k > bound || (equal && equal_before + (int)e < need));
      const bool source = kept && j >= budget, target = j < L && !kept && j < budget;
      equal_before += (int)all;
      const uint32_t at = block_prefix((source ? 1u : 0u) | (target ? 65536u : 0u), red, all);
      const int si = source_before + (int)(at & 65535u), ti = target_before + (int)(at >> 16);
      if (source && si < a.max_moves) sources[si] = j;
      if (target && ti < a.max_moves) targets[ti] = j;
      source_before += (int)(all & 65535u);
      target_before += (int)(all >> 16);
    }
    moves = source_before;
    if (moves > a.max_moves && threadIdx.x == 0) atomicExch(&g_key_eviction_error, 1);
  }
  for (int i = moves + threadIdx.x; i < a.max_moves; i += EV_THREADS) sources[i] = targets[i] = -1;
}

struct MoveArgs {
  void* pages;              // [n_pages, 2, nkv, page_size, d]
  float* scores;
  int* births;
  const int* block_table;
  const int* sources;
  const int* targets;
  int bt_stride, table_width, nkv, page_size, n_pages, max_moves, row_bytes;
};

// V: what a lane carries at once
template <typename V>
__global__ void move_keys_kernel(const MoveArgs a) {
  pdl_prologue();
  const int lane = threadIdx.x & 31, kvh = blockIdx.y, seq = blockIdx.z;
  const int i = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (i >= a.max_moves) return;
  const size_t entry = ((size_t)seq * a.nkv + kvh) * a.max_moves + i;
  const int source = a.sources[entry], target = a.targets[entry];
  if (source < 0 || target < 0 || source / a.page_size >= a.table_width || target / a.page_size >= a.table_width) return;
  const int* table = a.block_table + (size_t)seq * a.bt_stride;
  const int from = table[source / a.page_size], to = table[target / a.page_size];
  if (from < 0 || from >= a.n_pages || to < 0 || to >= a.n_pages) return;
  const int x = source % a.page_size, y = target % a.page_size, per_row = a.row_bytes / (int)sizeof(V);
  for (int c = lane; c < 2 * per_row; c += 32) {
    const int plane = c >= per_row, at = c - plane * per_row;
    const V* src = (const V*)((const char*)a.pages + ((((size_t)from * 2 + plane) * a.nkv + kvh) * a.page_size + x) * a.row_bytes);
    V* dst = (V*)((char*)a.pages + ((((size_t)to * 2 + plane) * a.nkv + kvh) * a.page_size + y) * a.row_bytes);
    dst[at] = src[at];
  }
  if (lane == 0) {
    const size_t s = ((size_t)from * a.nkv + kvh) * a.page_size + x, t = ((size_t)to * a.nkv + kvh) * a.page_size + y;
    a.scores[t] = a.scores[s];
    a.births[t] = a.births[s];
  }
}

}  // namespace

// Reads and clears the error word (0: none).  Synchronises the device.
NHV_API int nhv_key_eviction_error() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_key_eviction_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(g_key_eviction_error, &zero, sizeof(int));
  return v;
}
NHV_API void* nhv_key_eviction_error_word() {
  void* p = nullptr;
  return cudaGetSymbolAddress(&p, g_key_eviction_error) == cudaSuccess ? p : nullptr;
}

NHV_API int nhv_select_keys(int* sources, int* targets, const float* scores, const int* births, const int* block_table, int bt_stride,
                            const int* kv_len, const int* seen, const int* budgets, int n_seqs, int max_kv_len, int nkv, int page_size,
                            int n_pages, int max_moves, int keep_first, int keep_recent, cudaStream_t stream) {
  NHV_REQUIRE(nkv > 0 && page_size > 0 && n_pages > 0 && bt_stride >= 0, "choice of keys: bad page geometry");
  NHV_REQUIRE(n_seqs >= 0 && n_seqs <= 65535 && max_kv_len >= 0 && max_moves >= 0, "choice of keys: %d requests, %d keys, %d moves", n_seqs,
              max_kv_len, max_moves);
  NHV_REQUIRE(keep_first >= 0 && keep_recent >= 0, "choice of keys: kept first and recent keys are counted from 0");
  if (n_seqs == 0 || max_moves == 0) return 0;
  const ChoiceArgs a{scores, births, block_table, kv_len, seen, budgets, sources, targets, bt_stride, nkv, page_size, n_pages, max_moves,
                     keep_first, keep_recent, max_kv_len};
  NHV_CUDA(nhv_launch(select_keys_kernel, dim3(nkv, n_seqs), EV_THREADS, 0, stream, a), "choice of keys");
  return 0;
}

NHV_API int nhv_move_keys(void* kv_pages, float* scores, int* births, const int* block_table, int bt_stride, int table_width,
                          const int* sources, const int* targets, int n_seqs, int nkv, int page_size, int n_pages, int max_moves,
                          int row_bytes, cudaStream_t stream) {
  NHV_REQUIRE(nkv > 0 && nkv <= 65535 && page_size > 0 && n_pages > 0 && bt_stride >= table_width, "moves of keys: bad page geometry");
  NHV_REQUIRE(n_seqs >= 0 && n_seqs <= 65535 && max_moves >= 0 && row_bytes > 0 && row_bytes % 2 == 0, "moves of keys: %d requests, %d moves, rows of %d bytes",
              n_seqs, max_moves, row_bytes);
  if (n_seqs == 0 || max_moves == 0) return 0;
  const MoveArgs a{kv_pages, scores, births, block_table, sources, targets, bt_stride, table_width, nkv, page_size, n_pages, max_moves, row_bytes};
  const dim3 grid((max_moves + 7) / 8, nkv, n_seqs);
  if (row_bytes % 16 == 0 && (uintptr_t)kv_pages % 16 == 0)
    NHV_CUDA(nhv_launch(move_keys_kernel<uint4>, grid, 256, 0, stream, a), "moves of keys");
  else
    NHV_CUDA(nhv_launch(move_keys_kernel<uint16_t>, grid, 256, 0, stream, a), "moves of keys");
  return 0;
}
