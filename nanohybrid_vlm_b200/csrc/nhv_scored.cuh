// What the kernels of attention with scored keys share: their arguments, and the passes behind a split over the keys.
#pragma once
#include <math.h>

#include "nhv_common.cuh"

constexpr float SA_LOG2E = 1.4426950408889634f;
constexpr int SA_MAX_D = 256;
constexpr int SA_MOST_SPLITS = 32;                        // parts of a request's keys in the rows' pass
constexpr size_t SA_MOST_SUMS = (size_t)1 << 28;          // floats of their sums (1 GiB)

struct ScoredArgs {
  const void* q;
  void* out;
  const void* pages;
  const float* scores;      // [n_pages, nkv, page_size], what the keys had
  float* scores_out;        // the same with this step's weights (may be scores itself)
  int* births;              // [n_pages, nkv, page_size] or null
  const int* positions;     // per new token, with births
  const int* block_table;
  const int* cu_q;
  const int* kv_len;
  const float* sinks;       // per query head, or null
  float* lse;               // [nkv][n_tokens * G]: log2 of a row's sum; +inf for a row that sees nothing
  int q_stride, out_stride, bt_stride, n_seqs, n_tokens, nq, nkv, d, page_size, n_pages;
  int max_keys;             // what the caller says of kv_len: no table is read beyond it
  int min_rows, max_rows;   // a kernel takes the requests whose new tokens times G lie in this range (both included)
  float scale, softcap;
};

__device__ __forceinline__ bool scored_takes(const ScoredArgs& a, int n) {
  const int rows = n * (a.nq / a.nkv);
  return rows >= a.min_rows && rows <= a.max_rows;
}

// The request of row tile `tile`, its tiles counted in tokens of `per_tile`; -1 behind the last one.
__device__ __forceinline__ int find_tile(const ScoredArgs& a, int per_tile, int& tile) {
  for (int s = 0; s < a.n_seqs; ++s) {
    const int n = a.cu_q[s + 1] - a.cu_q[s];
    if (!scored_takes(a, n)) continue;
    const int nt = (n + per_tile - 1) / per_tile;
    if (tile < nt) return s;
    tile -= nt;
  }
  return -1;
}

// The element of a key's row in the pages, or -1 where the request has no page for it.
__device__ __forceinline__ long long key_row(const ScoredArgs& a, int seq, int j, int kvh, int plane) {
  const int page = a.block_table[(size_t)seq * a.bt_stride + j / a.page_size];
  if (page < 0 || page >= a.n_pages) return -1;
  return ((((long long)page * 2 + plane) * a.nkv + kvh) * a.page_size + j % a.page_size) * a.d;
}

// A key's sum of weights goes to its score, and a new key's position to its birth.  `fresh`: j - (keys before this step).
__device__ __forceinline__ void store_weight(const ScoredArgs& a, int seq, int first, int kvh, int j, int fresh, float sum) {
  const int page = a.block_table[(size_t)seq * a.bt_stride + j / a.page_size];
  if (page < 0 || page >= a.n_pages) return;
  const size_t at = ((size_t)page * a.nkv + kvh) * a.page_size + j % a.page_size;
  a.scores_out[at] = (fresh >= 0 ? 0.f : a.scores[at]) + sum;
  if (fresh >= 0 && a.births) a.births[at] = a.positions[first + fresh];
}

__device__ __forceinline__ float scored_exp2(float x) {     // 2^x; -inf gives 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// A pair of bfloat16 with what is not finite taken out; `bad` says whether there was any.
__device__ __forceinline__ uint32_t finite_pair(uint32_t v, bool& bad) {
  const bool lo = (v & 0x7f80u) == 0x7f80u, hi = (v & 0x7f800000u) == 0x7f800000u;
  bad |= lo | hi;
  return (lo ? 0u : v & 0xffffu) | (hi ? 0u : v & 0xffff0000u);
}

// Parts of the two passes: the keys of a request cut for the rows' pass (`splits`), its rows cut for the keys' pass (`chunks`).
struct ScoredParts {
  float* o;                 // [splits][nkv][n_tokens * G][d], with splits > 1
  float* ml;                // [splits][nkv][n_tokens * G][2]: reference and sum, in log2 units
  float* w;                 // [n_seqs][nkv][chunks][keys], with chunks > 1
  size_t keys;              // places for keys of a (request, KV head)
  int splits, split_tiles;  // parts of a request's keys, tiles of keys of one part
  int chunks, chunk_tiles;  // parts of a request's rows, tiles of rows of one part
  int tile_rows, tile_keys; // of the keys' pass
};
// The tiles of rows [begin, end) of chunk `chunk` that see some key of the tile of keys at key0.
__device__ __forceinline__ void chunk_range(const ScoredParts& p, int n, int G, int total, int key0, int chunk, int& begin, int& end) {
  const int t = key0 - (total - n), first = t > 0 ? t * G / p.tile_rows : 0, tiles = (n * G + p.tile_rows - 1) / p.tile_rows;
  begin = first > chunk * p.chunk_tiles ? first : chunk * p.chunk_tiles;
  end = tiles < (chunk + 1) * p.chunk_tiles ? tiles : (chunk + 1) * p.chunk_tiles;
}
// Fills in splits and chunks and the scratch they take; `row_tile` and `key_tile`: of the rows' pass, which takes
// about `tile_cycles` for one of each; blocks that run at once in either pass.
size_t scored_parts(ScoredParts& p, int n_seqs, int n_tokens, int max_new, int max_keys, int nq, int nkv, int d, int row_tile, int key_tile,
                    double tile_cycles, int rows_at_once, int keys_at_once);
// The most scratch of any call of up to so many requests and tokens, and keys of a request.
size_t scored_most_parts(int n_seqs, int n_tokens, int max_keys, int nq, int nkv, int d, int tile_rows, int tile_keys, int keys_at_once);
void scored_place(ScoredParts& p, float* work, int n_tokens, int nq, int d);
int scored_join_rows(int dtype, const ScoredArgs& a, const ScoredParts& p, cudaStream_t stream);
int scored_join_keys(const ScoredArgs& a, const ScoredParts& p, cudaStream_t stream);

// ---- requests with few rows (scored_attention_short.cu): the keys are split over blocks, the scores kept for the second pass
struct ShortPlan {
  int rows;                 // rows kept per key: the most of a request, rounded up to 2
  int block_rows, row_blocks;       // rows of a block, blocks that share a request's rows
  int split_keys, splits;   // keys of a block, parts of a request's keys
  int cluster;              // blocks that finish a (request, KV head) in one launch, or 0
  int group;                // requests per pair of launches (the scores kept are bounded)
  size_t keys;              // places for keys of a (request, KV head)
  size_t floats;            // of scratch
  size_t smem;              // bytes of a block
};
// The most rows of a request that goes this way, and whether requests of up to `rows` rows can.
int scored_short_rows(int dtype, int d);
bool scored_short_takes(int dtype, int rows, int d);
ShortPlan scored_short_plan(int dtype, int n_seqs, int max_rows, int max_keys, int nkv, int d);
size_t scored_short_most(int dtype, int n_seqs, int max_keys, int G, int nkv, int d);      // floats, for any call of up to these sizes
// The requests with a.min_rows to a.max_rows rows: output, scores and births.  `work`: plan.floats floats.
int scored_short_launch(int dtype, ScoredArgs a, const ShortPlan& plan, float* work, cudaStream_t stream);

// ---- requests with many rows, bfloat16 (scored_attention_tcgen05.cu)
bool scored_long_takes(int dtype, int nq, int nkv, int d, int page_size, int q_stride, float scale);
size_t scored_long_plan(ScoredParts& p, int n_seqs, int n_tokens, int max_new, int max_keys, int nq, int nkv, int d);     // floats of scratch
size_t scored_long_most(int n_seqs, int n_tokens, int max_keys, int nq, int nkv, int d);
// Whether the pool's rows fit a copy's 32-bit coordinate and the tiles the grid.
bool scored_long_reaches(const ScoredParts& p, int n_seqs, int n_tokens, int nq, int nkv, int d, int page_size, int n_pages);
int scored_long_launch(ScoredArgs a, const ScoredParts& p, cudaStream_t stream);
