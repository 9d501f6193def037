// Dropping keys from a paged cache by the attention weight that they have gathered (their scores).
//
// The choice, per request and KV head.  The keys of the first `keep_first` positions and of the last `keep_recent` count as
// +inf, a score that is no number as less than any; the `budget` largest stay, of equal ones those in the lowest slots.  It is said
// as moves: the i-th kept slot at or above the budget is the source for the i-th dropped slot below it.  After the moves the request's
// keys fill the slots [0, budget), in no order, which attention does not need; births say which position a slot holds.
// Every source lies at or above the budget and every target below it, so the moves may run in any order, and may run twice.
//
//   choice: a cluster of up to eight blocks per (request, KV head), each with a run of its slots.  The scores become whole numbers
//     of the same order, read once and kept in shared memory.  Their budget-th largest is found from counts of 11, 11 and 10 bits,
//     each block counting its own and reading the others' counts through the cluster; then every warp goes over its own run of slots
//     three times, without a barrier inside: keys equal to the bound are counted, then sources and targets, then written.
//   moves: a warp for eight moves, whose loads are all sent before the first store: K row, V row, score and birth.
//
// What bounds them: the choice reads 8 bytes a key and is a chain of counts, meetings and prefix sums (64 requests of 2,304 keys and 8
// heads 19 us, eight of 20,000 to 40,000 keys 32 us, against 2 and 3 us of reading); the moves are bound by memory (137 MB in 28 us,
// 242 MB in 44 us, 4.9 and 5.5 TB/s of the 6.5 that a copy has).
#include "nhv_common.cuh"

namespace {

constexpr int EV_BINS = 2048, EV_MOST_BLOCKS = 8, EV_LIST = 1024;
constexpr int EV_MOST_KEPT = 40960;           // keys of a block that shared memory holds; longer runs are read again from the pages

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
  int page_shift;           // log2 of the page size, -1 if that is no whole number
  int blocks, kept;         // of a cluster; keys of a block that fit its shared memory
};

__device__ __forceinline__ uint32_t key_of(const ChoiceArgs& a, const int* table, int kvh, int j, int recent) {
  const int at = a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size, page = table[at];
  if (page < 0 || page >= a.n_pages) return 0u;
  const size_t slot = ((size_t)page * a.nkv + kvh) * a.page_size + (j - at * a.page_size);
  const int birth = a.births[slot];
  const float score = a.scores[slot];
  return birth < a.keep_first || birth >= recent ? ordered(INFINITY) : ordered(score);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// A word of this block's shared memory as block `rank` of the cluster has it.
__device__ __forceinline__ uint32_t peer_address(const int* mine, int rank) {
  uint32_t addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(addr) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
  return addr;
}
__device__ __forceinline__ int peer_word(const int* mine, int rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];\n" : "=r"(v) : "r"(peer_address(mine, rank)) : "memory");
  return v;
}
// The sum of a word over the blocks of the cluster.
__device__ __forceinline__ int cluster_total(const int* mine, int blocks) {
  if (blocks == 1) return *mine;
  int sum = 0;
#pragma unroll
  for (int r = 0; r < EV_MOST_BLOCKS; ++r) sum += r < blocks ? peer_word(mine, r) : 0;
  return sum;
}
// Inclusive prefix sum over a warp.
__device__ __forceinline__ int warp_prefix(int v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += y;
  }
  return v;
}

template <int EV_THREADS>
__global__ void __launch_bounds__(EV_THREADS, 1024 / EV_THREADS) select_keys_kernel(const ChoiceArgs a) {
  constexpr int EV_WARPS = EV_THREADS / 32;
  extern __shared__ uint32_t s_keys[];                // [kept]
  __shared__ int s_count[3][EV_BINS], s_coarse[3][64];      // s_coarse: sums of 32 bins
  __shared__ int s_warp[3][EV_WARPS];                 // per warp: equal keys, sources, targets
  __shared__ int s_total[2];                          // the block's sources and targets
  __shared__ int s_digit, s_need, s_equal;            // the bound's next bits, what is left of the budget, keys equal to the bound
  __shared__ int s_listed, s_list[EV_LIST];           // slots that agree with the bound's first bits
  pdl_prologue();
  const int kvh = blockIdx.y, seq = blockIdx.z, rank = (int)cluster_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int L = min(a.kv_len[seq], a.max_keys), budget = max(0, a.budgets[seq]), recent = a.seen[seq] - a.keep_recent;
  const int* table = a.block_table + (size_t)seq * a.bt_stride;
  int* sources = a.sources + ((size_t)seq * a.nkv + kvh) * a.max_moves;
  int* targets = a.targets + ((size_t)seq * a.nkv + kvh) * a.max_moves;
  if (L <= budget || budget == 0) {                   // nothing to drop, or nothing to keep: no moves (the whole cluster agrees)
    for (int i = rank * EV_THREADS + threadIdx.x; i < a.max_moves; i += a.blocks * EV_THREADS) sources[i] = targets[i] = -1;
    return;
  }
  // the block's run of slots, and the warp's within it, whole groups of 32
  const int per_block = (L + a.blocks * 32 - 1) / (a.blocks * 32) * 32, begin = min(L, rank * per_block), end = min(L, begin + per_block);
  const int per_warp = (end - begin + EV_THREADS - 1) / EV_THREADS * 32, w_begin = min(end, begin + warp * per_warp), w_end = min(end, w_begin + per_warp);
  for (int i = threadIdx.x; i < 3 * EV_BINS; i += EV_THREADS) (&s_count[0][0])[i] = 0;
  if (threadIdx.x == 0) s_listed = 0;
  // eight slots a thread at once: their pages, then their births and scores, are asked for together
  for (int j0 = begin + threadIdx.x; j0 < min(end, begin + a.kept); j0 += 8 * EV_THREADS) {
    int page[8], birth[8];
    float score[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int j = j0 + u * EV_THREADS;
      page[u] = j < end ? table[a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size] : -1;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int j = j0 + u * EV_THREADS;
      const bool there = page[u] >= 0 && page[u] < a.n_pages;
      const size_t slot = ((size_t)(there ? page[u] : 0) * a.nkv + kvh) * a.page_size + (a.page_shift >= 0 ? j & (a.page_size - 1) : j % a.page_size);
      birth[u] = a.births[slot];
      score[u] = there ? a.scores[slot] : NAN;
      if (!there) birth[u] = 0x80000000;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int j = j0 + u * EV_THREADS;
      const bool held = page[u] >= 0 && page[u] < a.n_pages && (birth[u] < a.keep_first || birth[u] >= recent);
      if (j < min(end, begin + a.kept)) s_keys[j - begin] = held ? ordered(INFINITY) : ordered(score[u]);
    }
  }
  auto key_at = [&](int j) { return j - begin < a.kept ? s_keys[j - begin] : key_of(a, table, kvh, j, recent); };
  __syncthreads();

  // the bound: the budget-th largest; `need`: how many of the keys that agree with it so far are kept
  uint32_t bound = 0, mask = 0;
  int need = budget;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : EV_BINS;
    if (pass == 0) {
#pragma unroll 4
      for (int j0 = begin; j0 < end; j0 += EV_THREADS) {
        const int j = j0 + threadIdx.x;
        // lanes that agree, as the kept keys at a request's end do, are counted at once
        const uint32_t digit = j < end ? key_at(j) >> 21 : 0xffffffffu;
        int same;
        __match_all_sync(0xffffffffu, digit, &same);
        if (j < end && (!same || lane == 0)) atomicAdd(&s_count[0][digit], same ? 32 : 1);
      }
    } else if (pass == 1 || s_listed > EV_LIST) {
      // few keys agree with the first bits: those are noted, and the last pass looks at them alone
#pragma unroll 4
      for (int j = begin + threadIdx.x; j < end; j += EV_THREADS) {
        const uint32_t k = key_at(j);
        if ((k & mask) == bound) {
          atomicAdd(&s_count[pass][k >> shift & (bins - 1)], 1);
          if (pass == 1) {
            const int i = atomicAdd(&s_listed, 1);
            if (i < EV_LIST) s_list[i] = j;
          }
        }
      }
    } else {
      for (int i = threadIdx.x; i < s_listed; i += EV_THREADS) {
        const uint32_t k = key_at(s_list[i]);
        if ((k & mask) == bound) atomicAdd(&s_count[pass][k & (bins - 1)], 1);
      }
    }
    __syncthreads();
    // sums of 32 bins first, so that little is read from the other blocks (all 2,048 counts of eight blocks took 40 us a pass);
    // bins a pass does not use count nothing
    for (int c = warp; c < 64; c += EV_WARPS) {
      const int sum = __reduce_add_sync(0xffffffffu, s_count[pass][c * 32 + lane]);
      if (lane == 0) s_coarse[pass][c] = sum;
    }
    cluster_sync();
    if (warp == 0) {
      // from the highest down: the two groups of a lane, then the bins of the group in which the count reaches `need`
      const int c1 = cluster_total(&s_coarse[pass][63 - 2 * lane], a.blocks), c0 = cluster_total(&s_coarse[pass][62 - 2 * lane], a.blocks);
      int upto = warp_prefix(c1 + c0);
      int at = __ffs(__ballot_sync(0xffffffffu, upto >= need)) - 1;
      const int above_pair = __shfl_sync(0xffffffffu, upto - c1 - c0, at), upper = __shfl_sync(0xffffffffu, c1, at);
      const bool second = above_pair + upper < need;
      const int group = 63 - 2 * at - (second ? 1 : 0), above = above_pair + (second ? upper : 0);
      const int mine = cluster_total(&s_count[pass][group * 32 + 31 - lane], a.blocks);
      upto = above + warp_prefix(mine);
      at = __ffs(__ballot_sync(0xffffffffu, upto >= need)) - 1;
      if (lane == at) {
        s_digit = group * 32 + 31 - at;
        s_need = need - (upto - mine);
        s_equal = mine;
      }
    }
    __syncthreads();
    bound |= (uint32_t)s_digit << shift;
    need = s_need;
    mask |= (uint32_t)(bins - 1) << shift;
  }

  // Keys above the bound stay, and the first `need` of those equal to it: all of them unless a tie goes across the bound, for which
  // the equal keys before each warp's run are counted.
  const bool tie = s_equal > need;
  const unsigned lower = (1u << lane) - 1u;
  int equal_before = 0;
  if (tie) {
    int equal = 0;
    for (int j = w_begin + lane; j - lane < w_end; j += 32) equal += __popc(__ballot_sync(0xffffffffu, j < w_end && key_at(j) == bound));
    if (lane == 0) s_warp[0][warp] = equal;
    __syncthreads();
    for (int r = 0; r < rank; ++r) equal_before += peer_word(&s_count[2][bound & 1023u], r);
    for (int w = 0; w < warp; ++w) equal_before += s_warp[0][w];
  }
  // of 32 slots from j0 on: those that are kept at or above the budget, and those dropped below it
  auto moves_of = [&](int j0, int& e, unsigned& src, unsigned& dst) {
    const int j = j0 + lane;
    const bool in = j < w_end;
    const uint32_t k = in ? key_at(j) : 0u;
    bool stays = in && k >= bound;
    if (tie) {
      const unsigned eq = __ballot_sync(0xffffffffu, in && k == bound);
      stays = stays && (k != bound || e + __popc(eq & lower) < need);
      e += __popc(eq);
    }
    src = __ballot_sync(0xffffffffu, stays && j >= budget);
    dst = __ballot_sync(0xffffffffu, in && !stays && j < budget);
  };
  int n_source = 0, n_target = 0, e = equal_before;
  unsigned src, dst;
#pragma unroll 4
  for (int j0 = w_begin; j0 < w_end; j0 += 32) {
    moves_of(j0, e, src, dst);
    n_source += __popc(src);
    n_target += __popc(dst);
  }
  if (lane == 0) {
    s_warp[1][warp] = n_source;
    s_warp[2][warp] = n_target;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    int sum = 0;
    for (int w = 0; w < EV_WARPS; ++w) sum += s_warp[1 + threadIdx.x][w];
    s_total[threadIdx.x] = sum;
  }
  cluster_sync();
  int at_source = 0, at_target = 0, moves = 0;
  for (int r = 0; r < a.blocks; ++r) {
    const int x = r == rank ? s_total[0] : peer_word(&s_total[0], r);
    if (r < rank) {
      at_source += x;
      at_target += peer_word(&s_total[1], r);
    }
    moves += x;
  }
  for (int w = 0; w < warp; ++w) {
    at_source += s_warp[1][w];
    at_target += s_warp[2][w];
  }
  e = equal_before;
  for (int j0 = w_begin; j0 < w_end; j0 += 32) {
    moves_of(j0, e, src, dst);
    const int si = at_source + __popc(src & lower), ti = at_target + __popc(dst & lower);
    if ((src >> lane & 1u) && si < a.max_moves) sources[si] = j0 + lane;
    if ((dst >> lane & 1u) && ti < a.max_moves) targets[ti] = j0 + lane;
    at_source += __popc(src);
    at_target += __popc(dst);
  }
  if (moves > a.max_moves && threadIdx.x == 0 && rank == 0) atomicExch(&g_key_eviction_error, 1);
  for (int i = moves + rank * EV_THREADS + threadIdx.x; i < a.max_moves; i += a.blocks * EV_THREADS) sources[i] = targets[i] = -1;
  cluster_sync();                                     // no block leaves while another reads its counts
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

constexpr int MV_WARPS = 8, MV_MOVES = 8;      // moves of a warp

// V: what a lane carries at once.
template <typename V>
__global__ void __launch_bounds__(MV_WARPS * 32) move_keys_kernel(const MoveArgs a) {
  pdl_prologue();
  const int lane = threadIdx.x & 31, kvh = blockIdx.y, seq = blockIdx.z;
  const int i0 = (blockIdx.x * MV_WARPS + (threadIdx.x >> 5)) * MV_MOVES;
  if (i0 >= a.max_moves) return;
  // a lane per move looks up where it goes from and to: slots of the scores, which are rows of the key plane but for the page's planes
  long long from = -1, to = -1;
  if (lane < MV_MOVES && i0 + lane < a.max_moves) {
    const size_t entry = ((size_t)seq * a.nkv + kvh) * a.max_moves + i0 + lane;
    const int source = a.sources[entry], target = a.targets[entry];
    if (source >= 0 && target >= 0 && source / a.page_size < a.table_width && target / a.page_size < a.table_width) {
      const int* table = a.block_table + (size_t)seq * a.bt_stride;
      const int x = table[source / a.page_size], y = table[target / a.page_size];
      if (x >= 0 && x < a.n_pages && y >= 0 && y < a.n_pages) {
        const long long s = ((long long)x * a.nkv + kvh) * a.page_size + source % a.page_size;
        const long long t = ((long long)y * a.nkv + kvh) * a.page_size + target % a.page_size;
        const float score = a.scores[s];
        const int birth = a.births[s];
        a.scores[t] = score;
        a.births[t] = birth;
        from = s + (long long)x * a.nkv * a.page_size;
        to = t + (long long)y * a.nkv * a.page_size;
      }
    }
  }
  if (!__any_sync(0xffffffffu, from >= 0)) return;
  const int per_row = a.row_bytes / (int)sizeof(V);
  const long long plane = (long long)a.nkv * a.page_size;
  V* pages = (V*)a.pages;
  for (int c0 = 0; c0 < 2 * per_row; c0 += 32) {
    const int c = c0 + lane;
    const bool in = c < 2 * per_row, value = c >= per_row;
    V v[MV_MOVES];
#pragma unroll
    for (int k = 0; k < MV_MOVES; ++k) {
      const long long row = __shfl_sync(0xffffffffu, from, k);
      if (row >= 0 && in) v[k] = pages[(row + (value ? plane : 0)) * per_row + (value ? c - per_row : c)];
    }
#pragma unroll
    for (int k = 0; k < MV_MOVES; ++k) {
      const long long row = __shfl_sync(0xffffffffu, to, k);
      if (row >= 0 && in) pages[(row + (value ? plane : 0)) * per_row + (value ? c - per_row : c)] = v[k];
    }
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
  NHV_REQUIRE(n_seqs >= 0 && n_seqs <= 65535 && max_kv_len >= 0 && max_moves >= 0 && nkv <= 65535, "choice of keys: %d requests, %d keys, %d moves", n_seqs,
              max_kv_len, max_moves);
  NHV_REQUIRE(keep_first >= 0 && keep_recent >= 0, "choice of keys: kept first and recent keys are counted from 0");
  if (n_seqs == 0) return 0;                          // without room for moves the kernel still says whether some were needed
  ChoiceArgs a{scores, births, block_table, kv_len, seen, budgets, sources, targets, bt_stride, nkv, page_size, n_pages, max_moves,
               keep_first, keep_recent, max_kv_len};
  a.page_shift = -1;
  for (int k = 0; k < 31; ++k)
    if (page_size == 1 << k) a.page_shift = k;
  // blocks of a cluster: as many as fill the SMs (two blocks each), but a thousand slots a block at least
  const long long pairs = (long long)n_seqs * nkv;
  a.blocks = 1;
  while (a.blocks < EV_MOST_BLOCKS && pairs * a.blocks * 2 <= 2 * 148 * 2 && max_kv_len > a.blocks * 1024) a.blocks *= 2;
  const int per_block = (max_kv_len + a.blocks * 32 - 1) / (a.blocks * 32) * 32;
  a.kept = per_block < EV_MOST_KEPT ? per_block : EV_MOST_KEPT;
  static std::atomic<uint64_t> small_done{0}, done{0};
  const dim3 grid(a.blocks, nkv, n_seqs);
  if (per_block <= 8192) {          // four blocks an SM
    NHV_CUDA(nhv_allow_smem((const void*)select_keys_kernel<256>, EV_MOST_KEPT * 4, small_done), "choice of keys");
    NHV_CUDA(nhv_launch_cluster(select_keys_kernel<256>, grid, 256, (size_t)a.kept * 4, stream, a.blocks, a), "choice of keys");
  } else {
    NHV_CUDA(nhv_allow_smem((const void*)select_keys_kernel<512>, EV_MOST_KEPT * 4, done), "choice of keys");
    NHV_CUDA(nhv_launch_cluster(select_keys_kernel<512>, grid, 512, (size_t)a.kept * 4, stream, a.blocks, a), "choice of keys");
  }
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
  const dim3 grid((max_moves + MV_WARPS * MV_MOVES - 1) / (MV_WARPS * MV_MOVES), nkv, n_seqs);
  if (row_bytes % 16 == 0 && (uintptr_t)kv_pages % 16 == 0)
    NHV_CUDA(nhv_launch(move_keys_kernel<uint4>, grid, MV_WARPS * 32, 0, stream, a), "moves of keys");
  else
    NHV_CUDA(nhv_launch(move_keys_kernel<uint16_t>, grid, MV_WARPS * 32, 0, stream, a), "moves of keys");
  return 0;
}
