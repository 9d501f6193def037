// Attention with scored keys for requests that bring few rows (a row: a new token and a query head of one KV head), 8 to 32 of them at
// most (scored_short_rows): decoded tokens, drafts.  All the work is to read the keys and values once.
//
// First kernel: a block per (part of a request's keys, up to 24 of its rows, KV head, request), its warps independent of one another;
// blocks for other rows of the same keys find them in L2.  A warp takes 16 keys at a time straight from the pages into registers and
// forms S^T = K Q^T (m16n8k16, the 16 keys as M, up to 8 rows as N) and O^T += V^T P^T.  No shared memory is between the pages and the
// products: which element of a head stands at which index of the product is free as long as both operands agree, so a lane takes 16
// consecutive bytes of a row and its registers are the fragment as they are.  For V^T two keys' elements have to share a register, which
// one byte permutation each does.  The next keys' loads are sent as soon as the products have used the registers; the next tile's page is
// looked up one tile ahead.
//   P goes into the second product as two bfloat16 parts, its first 8 bits and what they leave (an error of 2^-15 where one part has
//   2^-8): the tensor pipe is idle most of the time here.  Neither part is negative, and the second none only where P is: an infinite
//   value times P is as infinite in parts as whole.  With more than 16 rows the pipe is not idle, and P has one part, as in the tcgen05
//   kernels (error of the output against 64 bits 2.3e-3, with two parts 1.7e-3, which is the output's own rounding).
//   The running maximum moves only when it grows by more than 2^8, so that most tiles leave the sums as they are.
//   The warps' sums meet in shared memory; the block leaves one partial sum (fp32) and the scores of its keys.
// Second kernel, or the same blocks as a cluster where few suffice: the parts' sums are joined, blocks of the output's elements and
// blocks of keys for the weights: a thread per key adds exp2(score - log-sum) over the rows.  Two kernels instead of one that reads the
// keys twice: a score is 4 bytes a row where a key is 2 d.
//
// What bounds it is reading the pages: 64 decoded tokens over 1,200 to 2,304 keys each (474 MB), 32 heads on 8 of 128, 99 us in both
// kernels, of them 85 in the first at 5.6 TB/s; three over 65,000 to 98,000 keys 173 to 181 us.  With 20 rows a request (drafts) it is
// the instructions of the products and exponentials, with two blocks an SM to hide them: 121 us for 311 MB.
//
// A key out of sight may hold anything: its score is replaced, its value not loaded.  Where only some of a request's rows see a key
// (several new tokens), what is not finite in the values is left out of the second product and given to the rows that see it.
#include "nhv_scored.cuh"

namespace {

constexpr int SH_WARPS = 4, SH_THREADS = SH_WARPS * 32, FIN_THREADS = 256, FIN_KEYS = 4;
constexpr int SH_MOST_ROWS = 24, SH_MOST_CLUSTER = 8;
constexpr int SH_MOST_SMEM = 100 * 1024;
constexpr float SH_GROW = 8.0f;                  // log2 units
constexpr size_t SH_MOST_SCORES = (size_t)1 << 28;        // floats of scores kept at once (1 GiB)

struct ShortArgs {
  ScoredArgs a;
  NhvScoreCap cap;
  float* kept;              // [group][nkv][keys][rows] scores in log2 units
  float* part_o;            // [group][nkv][splits][rows][d]
  float* part_ml;           // [group][nkv][splits][rows][2]: reference and sum
  size_t keys;
  int rows, block_rows, row_blocks, split_keys, splits, first_seq;
  int cluster;              // blocks that finish a (request, KV head) among themselves; 0: another kernel does
};

__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {      // an 8 x 8 tile of 16-bit numbers over the warp
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float low_of(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high_of(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// The weight of keys j0, j0 + step, .. from their kept scores, where some row's sum is no number: a row that does not see a key adds nothing.
__device__ __forceinline__ void careful_weights(const ScoredArgs& a, const float* kept, int stride, const float* lse, int rows, int seq, int first, int kvh,
                                                int j0, int step, int end, int old) {
#pragma unroll 1
  for (int j = j0; j < end; j += step) {
    float sum = 0.f;
#pragma unroll 1
    for (int r = 0; r < rows; ++r) {
      const float x = kept[(size_t)j * stride + r];
      sum += x == -INFINITY ? 0.f : scored_exp2(x - lse[r]);
    }
    store_weight(a, seq, first, kvh, j, j - old, sum);
  }
}

// The sums of a block's warps (in shared memory, rows of `row_len`) joined: the block's part, d floats a row, and its references and sums.
__device__ __forceinline__ void join_warps(const ShortArgs& w, const float* so, const float* sml, int row_len, float* part_o, float* part_ml, int rows, int d) {
  for (int i = threadIdx.x; i < rows * (d / 2); i += SH_THREADS) {
    const int r = i / (d / 2), c = 2 * (i - r * (d / 2));
    float ref = -INFINITY;
#pragma unroll
    for (int k = 0; k < SH_WARPS; ++k) ref = fmaxf(ref, sml[(k * w.block_rows + r) * 2]);
    const float use = ref == -INFINITY ? 0.f : ref;
    float sum = 0.f;
    float2 v = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < SH_WARPS; ++k) {
      const float f = scored_exp2(sml[(k * w.block_rows + r) * 2] - use);
      const float2 x = *reinterpret_cast<const float2*>(so + (k * w.block_rows + r) * row_len + c);
      sum = fmaf(f, sml[(k * w.block_rows + r) * 2 + 1], sum);
      v.x = fmaf(f, x.x, v.x);
      v.y = fmaf(f, x.y, v.y);
    }
    *reinterpret_cast<float2*>(part_o + r * d + c) = v;
    if (c == 0) *reinterpret_cast<float2*>(part_ml + r * 2) = make_float2(ref, sum);
  }
}

__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// This block's shared memory as block `rank` of the cluster has it.
__device__ __forceinline__ uint32_t peer_address(const float* mine, int rank) {
  uint32_t addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(addr) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
  return addr;
}
__device__ __forceinline__ float2 peer_load2(const float* mine, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "r"(peer_address(mine, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 peer_load4(const float* mine, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer_address(mine, rank)) : "memory");
  return v;
}

// Where a block's shared memory holds what: the warps' sums, the block's part, its keys' scores (in clusters).
__host__ __device__ __forceinline__ int short_sums(int block_rows, int d) { return SH_WARPS * block_rows * (d + 6); }
__host__ __device__ __forceinline__ int short_part(int block_rows, int d) { return (block_rows * (d + 2) + 3) / 4 * 4; }

// The keys of block `split`: as the plan cut the longest request, or, in a cluster, an even share of its own request's.
__device__ __forceinline__ void split_range(const ShortArgs& w, int split, int total, int& begin, int& end) {
  int keys = w.split_keys;
  if (w.cluster) keys = (total + w.cluster * 64 - 1) / (w.cluster * 64) * 64;
  begin = split * keys;
  end = min(total, begin + keys);
}

// What the second kernel does, by the blocks of a cluster: every block joins the parts' references and sums, makes its share of the
// output from all parts and the weights of its own keys.  All threads of all blocks come here.
template <typename T>
__device__ __forceinline__ void finish_in_cluster(const ShortArgs& w, float* smem, int row_len, int seq, int kvh, int first, int n, int total, int begin, int end) {
  __shared__ float s_f[SH_MOST_ROWS][SH_MOST_CLUSTER], s_lse[SH_MOST_ROWS];       // a part's factor in a row of the output; the row's log-sum
  const ScoredArgs& a = w.a;
  const int d = a.d, G = a.nq / a.nkv, R = min(n * G, w.block_rows), warp = threadIdx.x >> 5, lane = threadIdx.x & 31, old = total - n;
  float* part_o = smem + short_sums(w.block_rows, d);
  float* part_ml = part_o + w.block_rows * d;
  const float* kept = part_o + short_part(w.block_rows, d);
  join_warps(w, smem, smem + SH_WARPS * w.block_rows * row_len, row_len, part_o, part_ml, R, d);
  cluster_arrive();
  // the keys' places and what they had, asked for before the parts are there
  int page[FIN_KEYS];
  float had[FIN_KEYS];
  auto ask = [&](int j0) {
#pragma unroll
    for (int k = 0; k < FIN_KEYS; ++k) {
      const int j = j0 + k * SH_THREADS;
      page[k] = j < end ? a.block_table[(size_t)seq * a.bt_stride + j / a.page_size] : -1;
      if (page[k] >= a.n_pages) page[k] = -1;
      had[k] = 0.f;
      if (page[k] >= 0 && j < old) had[k] = a.scores[((size_t)page[k] * a.nkv + kvh) * a.page_size + j % a.page_size];
    }
  };
  ask(begin + threadIdx.x);
  cluster_wait();
  bool odd = false;                               // some row's sum is no number
  for (int r = warp; r < R; r += SH_WARPS) {
    const float sink = a.sinks ? a.sinks[kvh * G + r % G] * SA_LOG2E : -INFINITY;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < w.cluster) ml = peer_load2(part_ml + 2 * r, lane);
    const float ref = fmaxf(sink, warp_max(ml.x)), use = ref == -INFINITY ? 0.f : ref;
    const float f = scored_exp2(ml.x - use), sum = warp_sum(f * ml.y) + scored_exp2(sink - use);
    if (lane < w.cluster) s_f[r][lane] = sum == 0.f ? 0.f : f * (1.0f / sum);
    if (lane == 0) s_lse[r] = sum == 0.f ? INFINITY : use + log2f(sum);
    odd |= sum != sum;
  }
  odd = __syncthreads_or(odd);
  for (int i = blockIdx.x * SH_THREADS + threadIdx.x; i < R * (d / 4); i += w.cluster * SH_THREADS) {
    const int r = i / (d / 4), c = 4 * (i - r * (d / 4));
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < SH_MOST_CLUSTER; ++k) {
      if (k >= w.cluster) break;
      const float f = s_f[r][k];
      const float4 x = peer_load4(part_o + r * d + c, k);
      v.x = fmaf(f, x.x, v.x); v.y = fmaf(f, x.y, v.y); v.z = fmaf(f, x.z, v.z); v.w = fmaf(f, x.w, v.w);
    }
    T* dst = (T*)a.out + (size_t)(first + r / G) * a.out_stride + (size_t)(kvh * G + r % G) * d + c;
    if (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = v;
    else *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(v.x, v.y), pack2(v.z, v.w));
  }
  cluster_arrive();                               // nothing of the others is read behind this
  if (odd) careful_weights(a, kept - (ptrdiff_t)begin * w.rows, w.rows, s_lse, R, seq, first, kvh, begin + threadIdx.x, SH_THREADS, end, old);
  for (int j0 = odd ? end : begin + threadIdx.x; j0 < end; j0 += FIN_KEYS * SH_THREADS) {
#pragma unroll
    for (int k = 0; k < FIN_KEYS; ++k) {
      const int j = j0 + k * SH_THREADS;
      if (page[k] < 0) continue;
      const float* x = kept + (size_t)(j - begin) * w.rows;
      float sum = 0.f;
      for (int r = 0; r < R; r += 2) {
        const float2 v = *reinterpret_cast<const float2*>(x + r);
        sum += scored_exp2(v.x - s_lse[r]);
        if (r + 1 < R) sum += scored_exp2(v.y - s_lse[r + 1]);
      }
      const size_t at = ((size_t)page[k] * a.nkv + kvh) * a.page_size + j % a.page_size;
      a.scores_out[at] = had[k] + sum;
      if (j >= old && a.births) a.births[at] = a.positions[first + j - old];
    }
    ask(j0 + FIN_KEYS * SH_THREADS);
  }
  cluster_wait();
}

// DB: blocks of 64 elements of a head; NT: blocks of 8 rows; BY16: pages hold a multiple of 16 keys.
template <int DB, int NT, bool BY16>
__global__ void __launch_bounds__(SH_THREADS, DB * NT <= 2 ? 3 : 2) scored_short_kernel(const ShortArgs w) {
  constexpr int PARTS = NT <= 2 ? 2 : 1;          // of P
  extern __shared__ __align__(16) float smem[];                 // [warps][rows][d + 2] sums, then [warps][rows][2]
  const ScoredArgs& a = w.a;
  pdl_prologue();
  const int seq = w.first_seq + blockIdx.z, kvh = blockIdx.y, G = a.nq / a.nkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = a.cu_q[seq], n = a.cu_q[seq + 1] - first, total = min(a.kv_len[seq], a.max_keys), R = n * G, d = a.d;
  const int split = blockIdx.x / w.row_blocks, r0 = (blockIdx.x - split * w.row_blocks) * w.block_rows, RB = min(R - r0, w.block_rows);
  int begin, end;
  split_range(w, split, total, begin, end);
  if ((!w.cluster && (begin >= end || RB <= 0)) || !scored_takes(a, n)) return;
  const int ra = lane >> 2, rc = lane & 3;
  const __nv_bfloat16* q = (const __nv_bfloat16*)a.q;
  const __nv_bfloat16* pages = (const __nv_bfloat16*)a.pages;
  const int* table = a.block_table + (size_t)seq * a.bt_stride;
  const size_t v_plane = (size_t)a.nkv * a.page_size * d;

  // the product's B operand: row r0 + ra (+ 8), elements 32 i + 8 rc ..
  uint4 qf[NT][2 * DB];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = t * 8 + ra;
#pragma unroll
    for (int i = 0; i < 2 * DB; ++i) {
      const int e = 32 * i + 8 * rc;
      qf[t][i] = make_uint4(0, 0, 0, 0);
      if (r < RB && e < d) qf[t][i] = *reinterpret_cast<const uint4*>(q + (size_t)(first + (r0 + r) / G) * a.q_stride + (size_t)(kvh * G + (r0 + r) % G) * d + e);
    }
  }
  float o[NT][DB][4][4];                          // O^T: element 64 b + 8 ra + 2 u (+ 1), rows 2 rc (+ 1)
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t][0] = m[t][1] = -INFINITY;
    l[t][0] = l[t][1] = 0.f;
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int u = 0; u < 4; ++u) o[t][b][u][0] = o[t][b][u][1] = o[t][b][u][2] = o[t][b][u][3] = 0.f;
  }
  uint4 kr[2][2 * DB], vr[4][DB];
  // where a tile's keys lie: the page of the tile (BY16), looked up a tile ahead of its loads
  auto page_at = [&](int j) -> int {
    const int page = j < end ? table[j / a.page_size] : -1;
    return page < a.n_pages ? page : -1;
  };
  auto row_at = [&](int j, int tile_page, int tile_off, int in_tile) -> const __nv_bfloat16* {
    int page = tile_page, off = tile_off + in_tile;
    if (!BY16) {
      page = page_at(j);
      off = j % a.page_size;
    }
    return page < 0 || j >= end ? nullptr : pages + (((size_t)page * 2 * a.nkv + kvh) * a.page_size + off) * d;
  };
  // a tile whose keys are all there and whose heads fill the lanes is read without a check a key
  const bool full = BY16 && d == 64 * DB;
  auto load_keys = [&](int j0, int page, int off) {
    if (full && page >= 0 && j0 + 16 <= end) {
      const __nv_bfloat16* row = pages + (((size_t)page * 2 * a.nkv + kvh) * a.page_size + off + ra) * (64 * DB) + 8 * rc;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2 * DB; ++i) kr[h][i] = load16(row + h * 8 * 64 * DB + 32 * i);
      return;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __nv_bfloat16* row = row_at(j0 + ra + 8 * h, page, off, ra + 8 * h);
#pragma unroll
      for (int i = 0; i < 2 * DB; ++i) {
        const int e = 32 * i + 8 * rc;
        kr[h][i] = row && e < d ? load16(row + e) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  auto load_values = [&](int j0, int page, int off) {
    if (full && page >= 0 && j0 + 16 <= end) {
      const __nv_bfloat16* row = pages + v_plane + (((size_t)page * 2 * a.nkv + kvh) * a.page_size + off + 2 * rc) * (64 * DB) + 8 * ra;
#pragma unroll
      for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int b = 0; b < DB; ++b) vr[h][b] = load16(row + ((h & 1) + 8 * (h >> 1)) * 64 * DB + 64 * b);
      return;
    }
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const int in_tile = 2 * rc + (h & 1) + 8 * (h >> 1);
      const __nv_bfloat16* row = row_at(j0 + in_tile, page, off, in_tile);
#pragma unroll
      for (int b = 0; b < DB; ++b) {
        const int e = 64 * b + 8 * ra;
        vr[h][b] = row && e < d ? load16(row + v_plane + e) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  auto second_product = [&](const uint32_t (&p)[NT][PARTS][2]) {
#pragma unroll
    for (int b = 0; b < DB; ++b) {
      const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&vr[0][b]);
      const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&vr[1][b]);
      const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&vr[2][b]);
      const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&vr[3][b]);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t a0 = __byte_perm(v0[u], v1[u], 0x5410), a1 = __byte_perm(v0[u], v1[u], 0x7632);
        const uint32_t a2 = __byte_perm(v2[u], v3[u], 0x5410), a3 = __byte_perm(v2[u], v3[u], 0x7632);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          mma16816(o[t][b][u], a0, a1, a2, a3, p[t][0][0], p[t][0][1]);
          if (PARTS == 2) mma16816(o[t][b][u], a0, a1, a2, a3, p[t][PARTS - 1][0], p[t][PARTS - 1][1]);
        }
      }
    }
  };
  float* kept = w.cluster ? smem + short_sums(w.block_rows, d) + short_part(w.block_rows, d) - (ptrdiff_t)begin * w.rows
                          : w.kept + ((size_t)blockIdx.z * a.nkv + kvh) * w.keys * w.rows + r0;
  const float scale_log2 = w.cap.in != 0.f ? 1.0f : a.scale * SA_LOG2E;

  const int step = 16 * SH_WARPS;
  int odd_tile = -1;
  int j0 = RB > 0 ? begin + 16 * warp : end;      // a request that brings nothing keeps its scores
  int page = page_at(j0), off = BY16 ? j0 % a.page_size : 0;
  int page_next = page_at(j0 + step);
  if (j0 < end) {
    load_keys(j0, page, off);
    load_values(j0, page, off);
  }
  for (; j0 < end; j0 += step) {
    float s[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * DB; ++i) {
        mma16816(s[t], kr[0][i].x, kr[1][i].x, kr[0][i].y, kr[1][i].y, qf[t][i].x, qf[t][i].y);
        mma16816(s[t], kr[0][i].z, kr[1][i].z, kr[0][i].w, kr[1][i].w, qf[t][i].z, qf[t][i].w);
      }
    }
    const int at_page = page, off_next = BY16 ? (j0 + step) % a.page_size : 0;
    page = page_next;
    off = off_next;
    load_keys(j0 + step, page, off);
    page_next = page_at(j0 + 2 * step);

    // scores in log2 units; -inf for what a row does not see
    const bool edge = j0 + 15 > total - n;
    if (w.cap.in != 0.f) nhv_cap_tile<NT, true>(s, w.cap);
    bool grow = false;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][e] *= scale_log2;
      if (edge || (BY16 && at_page < 0) || !BY16 || j0 + 16 > end) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + ra + 8 * (e >> 1), r = t * 8 + 2 * rc + (e & 1);
          bool sees = j < end && r < RB && j <= total - n + (r0 + r) / G;
          if (BY16) sees = sees && at_page >= 0;
          else sees = sees && page_at(j) >= 0;
          if (!sees) s[t][e] = -INFINITY;
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) grow |= fmaxf(s[t][e], s[t][2 + e]) > m[t][e] + SH_GROW;       // over the lanes only where it does
      if (t * 8 + 2 * rc < RB) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (j0 + ra + 8 * h < end) *reinterpret_cast<float2*>(kept + (size_t)(j0 + ra + 8 * h) * w.rows + t * 8 + 2 * rc) = make_float2(s[t][2 * h], s[t][2 * h + 1]);
      }
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(s[t][e], s[t][2 + e]);
#pragma unroll
          for (int k = 4; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
          if (top > m[t][e] + SH_GROW) {
            const float alpha = scored_exp2(m[t][e] - top);            // 0 when the row had seen nothing
            m[t][e] = top;
            l[t][e] *= alpha;
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                o[t][b][u][e] *= alpha;
                o[t][b][u][2 + e] *= alpha;
              }
          }
        }
    }
    uint32_t p[NT][PARTS][2];                      // [first bits, what they leave][keys 0-7, 8-15], or [rounded]
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[e] = scored_exp2(s[t][2 * h + e] - (m[t][e] == -INFINITY ? 0.f : m[t][e]));
          l[t][e] += x[e];
        }
        if (PARTS == 2) {
          const uint32_t hi = __byte_perm(__float_as_uint(x[0]), __float_as_uint(x[1]), 0x7632);
          p[t][0][h] = transposed(hi);
          p[t][PARTS - 1][h] = transposed(pack2(fmaxf(x[0] - low_of(hi), x[0] * 0x1p-20f), fmaxf(x[1] - high_of(hi), x[1] * 0x1p-20f)));
        } else {
          p[t][0][h] = transposed(pack2(x[0], x[1]));
        }
      }
    if (!edge || n == 1) {
      second_product(p);
    } else {
      // some row does not see some key: what is not finite in the values comes behind the walk, to the rows that see it.  Such a tile
      // touches the request's last 32 keys, so a warp, which takes every fourth, meets one at most.
      bool odd = false;
#pragma unroll
      for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int b = 0; b < DB; ++b) {
          vr[h][b].x = finite_pair(vr[h][b].x, odd); vr[h][b].y = finite_pair(vr[h][b].y, odd);
          vr[h][b].z = finite_pair(vr[h][b].z, odd); vr[h][b].w = finite_pair(vr[h][b].w, odd);
        }
      if (__any_sync(0xffffffffu, odd)) odd_tile = j0;
      second_product(p);
    }
    load_values(j0 + step, page, off);
  }

  // the warps' sums joined
  const int row_len = d + 2;
  float* so = smem;
  float* sml = smem + SH_WARPS * w.block_rows * row_len;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = l[t][e];
#pragma unroll
      for (int k = 4; k < 32; k <<= 1) x += __shfl_xor_sync(0xffffffffu, x, k);
      const int r = t * 8 + 2 * rc + e;
      if (r < w.block_rows) {
        if (ra == 0) {
          sml[(warp * w.block_rows + r) * 2] = m[t][e];
          sml[(warp * w.block_rows + r) * 2 + 1] = x;
        }
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int at = 64 * b + 8 * ra + 2 * u;
            if (at < d) *reinterpret_cast<float2*>(so + (warp * w.block_rows + r) * row_len + at) = make_float2(o[t][b][u][e], o[t][b][u][2 + e]);
          }
      }
    }
  if (odd_tile >= 0) {
    // the values left out above, to this warp's sums: an element of the head a lane
    __syncwarp();
    for (int j = odd_tile; j < min(odd_tile + 16, end); ++j) {
      const int at = page_at(j), sees_from = max(0, (j - (total - n)) * G - r0);
      for (int c = lane; c < d && at >= 0; c += 32) {
        const float v = to_f32(pages[v_plane + (((size_t)at * 2 * a.nkv + kvh) * a.page_size + j % a.page_size) * d + c]);
        if (fabsf(v) < INFINITY) continue;
        for (int r = sees_from; r < RB; ++r) {
          const float ref = sml[(warp * w.block_rows + r) * 2];
          float& sum = so[(warp * w.block_rows + r) * row_len + c];
          sum = fmaf(scored_exp2(kept[(size_t)j * w.rows + r] - (ref == -INFINITY ? 0.f : ref)), v, sum);
        }
      }
    }
  }
  __syncthreads();
  if (w.cluster) {
    finish_in_cluster<__nv_bfloat16>(w, smem, row_len, seq, kvh, first, n, total, begin, end);
    return;
  }
  const size_t part = (((size_t)blockIdx.z * a.nkv + kvh) * w.splits + split) * w.rows + r0;
  join_warps(w, so, sml, row_len, w.part_o + part * d, w.part_ml + part * 2, RB, d);
}

// The same for float32, on the CUDA cores.  LPK lanes share a key, 4 EV / 4 elements each: a key's row is read in one piece, and
// what a row of the product needs of q and O stands in registers.  A warp takes U x 32 / LPK keys at a time; the lanes' parts of the U x RB
// scores are added by halves (a lane keeps half of its numbers and sends the other half), which costs about one shuffle a score and
// leaves each score in one lane, where its exponential is taken once.  P goes back to all lanes by a shuffle.
template <int LPK, int EV, int RB, bool BY_PAGE>
__global__ void __launch_bounds__(SH_THREADS, EV == 8 ? 2 : 3) scored_short_f32_kernel(const ShortArgs w) {
  extern __shared__ __align__(16) float smem[];                 // [warps][rows][d + 2] sums, then [warps][rows][2]
  constexpr int U = RB * EV >= 32 ? 4 : 8, KPI = 32 / LPK, BATCH = U * KPI, N = U * RB;
  constexpr int P = N > LPK ? N / LPK : 1, DUP = LPK > N ? LPK / N : 1;       // scores of a lane; lanes that hold the same one
  const ScoredArgs& a = w.a;
  pdl_prologue();
  const int seq = w.first_seq + blockIdx.z, kvh = blockIdx.y, G = a.nq / a.nkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = a.cu_q[seq], n = a.cu_q[seq + 1] - first, total = min(a.kv_len[seq], a.max_keys), R = n * G, d = a.d;
  const int split = blockIdx.x / w.row_blocks, r0 = (blockIdx.x - split * w.row_blocks) * w.block_rows, rows = min(R - r0, w.block_rows);
  int begin, end;
  split_range(w, split, total, begin, end);
  if ((!w.cluster && (begin >= end || rows <= 0)) || !scored_takes(a, n)) return;
  const int kk = lane / LPK, in_key = lane % LPK;
  const float* q = (const float*)a.q;
  const float* pages = (const float*)a.pages;
  const int* table = a.block_table + (size_t)seq * a.bt_stride;
  const size_t v_plane = (size_t)a.nkv * a.page_size * d;
  // elements 4 in_key .. of every block of 4 LPK
  float qf[RB][EV], o[RB][EV], m[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    m[r] = -INFINITY;
#pragma unroll
    for (int e = 0; e < EV; e += 4) {
      const int at = e * LPK + 4 * in_key;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < rows && at < d) x = *reinterpret_cast<const float4*>(q + (size_t)(first + (r0 + r) / G) * a.q_stride + (size_t)(kvh * G + (r0 + r) % G) * d + at);
      qf[r][e] = x.x; qf[r][e + 1] = x.y; qf[r][e + 2] = x.z; qf[r][e + 3] = x.w;
      o[r][e] = o[r][e + 1] = o[r][e + 2] = o[r][e + 3] = 0.f;
    }
  }
  float l[P], x[P];
#pragma unroll
  for (int i = 0; i < P; ++i) l[i] = 0.f;
  float4 kr[U][EV / 4], vr[U][EV / 4];
  auto row_at = [&](int j, int j0) -> const float* {
    if (j >= end) return nullptr;
    const int jp = BY_PAGE ? j0 : j, at = jp / a.page_size, page = table[at];
    if (page < 0 || page >= a.n_pages) return nullptr;
    return pages + (((size_t)page * 2 * a.nkv + kvh) * a.page_size + (j - at * a.page_size)) * d;
  };
  auto load = [&](float4 (&dst)[U][EV / 4], int j0, size_t plane) -> uint32_t {       // a bit for every u whose key is there
    if (BY_PAGE && j0 + BATCH <= end) {                     // a whole batch in one page: no check a key (552 -> 220 us for 64 requests)
      const float* row = row_at(j0, j0);
      if (row) {
        row += plane + (size_t)kk * d + 4 * in_key;
#pragma unroll
        for (int e = 0; e < EV / 4; ++e) {
          if (e * 4 * LPK + 4 * in_key < d) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const uint4 v = load16(row + (size_t)(u * KPI) * d + e * 4 * LPK);
              dst[u][e] = make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
            }
          } else {
#pragma unroll
            for (int u = 0; u < U; ++u) dst[u][e] = make_float4(0.f, 0.f, 0.f, 0.f);
          }
        }
        return 0xffffffffu;
      }
    }
    uint32_t there = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float* row = row_at(j0 + u * KPI + kk, j0);
      there |= row ? 1u << u : 0u;
#pragma unroll
      for (int e = 0; e < EV / 4; ++e) {
        const int at = e * 4 * LPK + 4 * in_key;
        dst[u][e] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row && at < d) {
          const uint4 v = load16(row + plane + at);
          dst[u][e] = make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
        }
      }
    }
    return there;
  };
  float* kept = w.cluster ? smem + short_sums(w.block_rows, d) + short_part(w.block_rows, d) - (ptrdiff_t)begin * w.rows
                          : w.kept + ((size_t)blockIdx.z * a.nkv + kvh) * w.keys * w.rows + r0;
  // the lane's scores: number i of the batch's U x RB is key i / RB, row i % RB
  const int i0 = in_key / DUP * P;
  const bool first_copy = in_key % DUP == 0;
  const int step = BATCH * SH_WARPS;
  int j0 = rows > 0 ? begin + BATCH * warp : end;     // a request that brings nothing keeps its scores
  uint32_t there = 0;
  if (j0 < end) {
    there = load(kr, j0, 0);
    load(vr, j0, v_plane);
  }
  for (; j0 < end; j0 += step) {
    float s[N];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        float t = 0.f;
#pragma unroll
        for (int e = 0; e < EV / 4; ++e) {
          t = fmaf(qf[r][4 * e], kr[u][e].x, t);
          t = fmaf(qf[r][4 * e + 1], kr[u][e].y, t);
          t = fmaf(qf[r][4 * e + 2], kr[u][e].z, t);
          t = fmaf(qf[r][4 * e + 3], kr[u][e].w, t);
        }
        s[u * RB + r] = t;
      }
    const uint32_t there_next = load(kr, j0 + step, 0);
    int count = N;
#pragma unroll
    for (int bit = LPK / 2; bit > 0; bit >>= 1) {
      if (count > 1) {
        count >>= 1;
#pragma unroll
        for (int i = 0; i < N / 2; ++i)
          if (i < count) {
            const bool upper = lane & bit;
            const float mine = upper ? s[i + count] : s[i], other = upper ? s[i] : s[i + count];
            s[i] = mine + __shfl_xor_sync(0xffffffffu, other, bit);
          }
      } else {
        s[0] += __shfl_xor_sync(0xffffffffu, s[0], bit);
      }
    }
    const bool edge = j0 + BATCH - 1 > total - n;
    bool grow = false;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int r = (i0 + i) % RB, j = j0 + (i0 + i) / RB * KPI + kk;
      float t = s[i] * a.scale;
      if (a.softcap > 0.f) t = a.softcap * tanhf(t / a.softcap);
      t *= SA_LOG2E;
      bool sees = (there >> (i0 + i) / RB & 1u) && r < rows;
      if (edge) sees = sees && j <= total - n + (r0 + r) / G;
      x[i] = sees ? t : -INFINITY;
      if (first_copy && j < end && r < rows) kept[(size_t)j * w.rows + r] = x[i];
      float ref = m[0];
#pragma unroll
      for (int k = 1; k < RB; ++k) ref = r == k ? m[k] : ref;
      grow |= x[i] > ref + SH_GROW;
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < P; ++i) top = fmaxf(top, (i0 + i) % RB == r ? x[i] : -INFINITY);
        top = warp_max(top);
        if (top > m[r] + SH_GROW) {
          const float alpha = scored_exp2(m[r] - top);
          m[r] = top;
#pragma unroll
          for (int i = 0; i < P; ++i)
            if ((i0 + i) % RB == r) l[i] *= alpha;
#pragma unroll
          for (int e = 0; e < EV; ++e) o[r][e] *= alpha;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int r = (i0 + i) % RB;
      float ref = m[0];
#pragma unroll
      for (int k = 1; k < RB; ++k) ref = r == k ? m[k] : ref;
      x[i] = scored_exp2(x[i] - (ref == -INFINITY ? 0.f : ref));
      l[i] += x[i];
    }
    auto second_product = [&](bool all) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          const int i = u * RB + r;
          const float p = __shfl_sync(0xffffffffu, x[i % P], kk * LPK + i / P * DUP);
          // where some row does not see some key, a value out of sight is left out: it may be no number
          if (all || (j0 + u * KPI + kk <= total - n + (r0 + r) / G)) {
#pragma unroll
            for (int e = 0; e < EV / 4; ++e) {
              o[r][4 * e] = fmaf(p, vr[u][e].x, o[r][4 * e]);
              o[r][4 * e + 1] = fmaf(p, vr[u][e].y, o[r][4 * e + 1]);
              o[r][4 * e + 2] = fmaf(p, vr[u][e].z, o[r][4 * e + 2]);
              o[r][4 * e + 3] = fmaf(p, vr[u][e].w, o[r][4 * e + 3]);
            }
          }
        }
    };
    if (!edge || n == 1) second_product(true);
    else second_product(false);
    load(vr, j0 + step, v_plane);
    there = there_next;
  }
  // the warps' sums joined
  const int row_len = d + 4;
  float* so = smem;
  float* sml = smem + SH_WARPS * w.block_rows * row_len;
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) sum += first_copy && (i0 + i) % RB == r ? l[i] : 0.f;
    sum = warp_sum(sum);
#pragma unroll
    for (int e = 0; e < EV; ++e)
#pragma unroll
      for (int bit = LPK; bit < 32; bit <<= 1) o[r][e] += __shfl_xor_sync(0xffffffffu, o[r][e], bit);
    if (r >= w.block_rows) continue;
    if (lane == 0) {
      sml[(warp * w.block_rows + r) * 2] = m[r];
      sml[(warp * w.block_rows + r) * 2 + 1] = sum;
    }
    if (kk == 0) {
#pragma unroll
      for (int e = 0; e < EV; e += 4) {
        const int at = e * LPK + 4 * in_key;
        if (at < d) *reinterpret_cast<float4*>(so + (warp * w.block_rows + r) * row_len + at) = make_float4(o[r][e], o[r][e + 1], o[r][e + 2], o[r][e + 3]);
      }
    }
  }
  __syncthreads();
  if (w.cluster) {
    finish_in_cluster<float>(w, smem, row_len, seq, kvh, first, n, total, begin, end);
    return;
  }
  const size_t part = (((size_t)blockIdx.z * a.nkv + kvh) * w.splits + split) * w.rows + r0;
  join_warps(w, so, sml, row_len, w.part_o + part * d, w.part_ml + part * 2, rows, d);
}

// Blocks [0, key_blocks): weights of `per_block` keys each, the others FIN_THREADS elements of the output each.
template <typename T>
__global__ void __launch_bounds__(FIN_THREADS) scored_short_finish_kernel(const ShortArgs w, const int key_blocks, const int per_block) {
  __shared__ float s_ref[32], s_inv[32], s_lse[32];
  const ScoredArgs& a = w.a;
  pdl_prologue();
  const int seq = w.first_seq + blockIdx.z, kvh = blockIdx.y, G = a.nq / a.nkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = a.cu_q[seq], n = a.cu_q[seq + 1] - first, total = min(a.kv_len[seq], a.max_keys), R = n * G, d = a.d;
  if (!scored_takes(a, n)) return;
  const bool output = blockIdx.x >= key_blocks;
  const int i = ((int)blockIdx.x - key_blocks) * FIN_THREADS + threadIdx.x;       // of the output
  if (output ? i - (int)threadIdx.x >= R * d : (int)blockIdx.x * per_block >= total) return;
  const int parts = (total + w.split_keys - 1) / w.split_keys;
  const size_t part = ((size_t)blockIdx.z * a.nkv + kvh) * w.splits * w.rows;
  bool odd = false;                               // some row's sum is no number
  for (int r = warp; r < R; r += FIN_THREADS / 32) {
    const float sink = a.sinks ? a.sinks[kvh * G + r % G] * SA_LOG2E : -INFINITY;
    float ref = sink, sum = 0.f;
    for (int k0 = 0; k0 < parts; k0 += 32) {
      float2 ml = make_float2(-INFINITY, 0.f);
      if (k0 + lane < parts) ml = *reinterpret_cast<const float2*>(w.part_ml + (part + (size_t)(k0 + lane) * w.rows + r) * 2);
      const float top = fmaxf(ref, warp_max(ml.x)), use = top == -INFINITY ? 0.f : top;
      sum = sum * scored_exp2(ref - use) + ml.y * scored_exp2(ml.x - use);
      ref = top;
    }
    const float use = ref == -INFINITY ? 0.f : ref;
    sum = warp_sum(sum) + scored_exp2(sink - use);
    if (lane == 0) {
      s_ref[r] = use;
      s_inv[r] = sum == 0.f ? 0.f : 1.0f / sum;
      s_lse[r] = sum == 0.f ? INFINITY : use + log2f(sum);
    }
    odd |= sum != sum;
  }
  odd = __syncthreads_or(odd);
  if (output) {
    if (i >= R * d) return;
    const int r = i / d, c = i - r * d;
    const float ref = s_ref[r];
    const float* ml = w.part_ml + (part + r) * 2;
    const float* po = w.part_o + (part + r) * d + c;
    const size_t step = w.rows;
    float v = 0.f;
#pragma unroll 8
    for (int k = 0; k < parts; ++k) v = fmaf(scored_exp2(ml[k * step * 2] - ref), po[k * step * d], v);
    ((T*)a.out)[(size_t)(first + r / G) * a.out_stride + (size_t)(kvh * G + r % G) * d + c] = from_f32<T>(v * s_inv[r]);
    return;
  }
  const float* kept = w.kept + ((size_t)blockIdx.z * a.nkv + kvh) * w.keys * w.rows;
  const int end = min(total, (int)(blockIdx.x + 1) * per_block), old = total - n, j0 = blockIdx.x * per_block + threadIdx.x;
  if (odd) {
    careful_weights(a, kept, w.rows, s_lse, R, seq, first, kvh, j0, FIN_THREADS, end, old);
    return;
  }
  // four keys a thread: their pages, their old scores and the rows' scores are asked for together
  int page[FIN_KEYS];
  size_t at[FIN_KEYS];
  float sum[FIN_KEYS];
#pragma unroll
  for (int k = 0; k < FIN_KEYS; ++k) {
    const int j = j0 + k * FIN_THREADS;
    page[k] = j < end ? a.block_table[(size_t)seq * a.bt_stride + j / a.page_size] : -1;
    sum[k] = 0.f;
  }
  if (w.rows % 4 == 0) {
#pragma unroll 2
    for (int r = 0; r < R; r += 4) {
      float4 x[FIN_KEYS];
#pragma unroll
      for (int k = 0; k < FIN_KEYS; ++k) x[k] = *reinterpret_cast<const float4*>(kept + (size_t)min(j0 + k * FIN_THREADS, end - 1) * w.rows + r);
#pragma unroll
      for (int k = 0; k < FIN_KEYS; ++k) {
        sum[k] += scored_exp2(x[k].x - s_lse[r]);
        if (r + 1 < R) sum[k] += scored_exp2(x[k].y - s_lse[r + 1]);
        if (r + 2 < R) sum[k] += scored_exp2(x[k].z - s_lse[r + 2]);
        if (r + 3 < R) sum[k] += scored_exp2(x[k].w - s_lse[r + 3]);
      }
    }
  } else {
#pragma unroll 2
    for (int r = 0; r < R; r += 2) {
      float2 x[FIN_KEYS];
#pragma unroll
      for (int k = 0; k < FIN_KEYS; ++k) x[k] = *reinterpret_cast<const float2*>(kept + (size_t)min(j0 + k * FIN_THREADS, end - 1) * w.rows + r);
#pragma unroll
      for (int k = 0; k < FIN_KEYS; ++k) {
        sum[k] += scored_exp2(x[k].x - s_lse[r]);
        if (r + 1 < R) sum[k] += scored_exp2(x[k].y - s_lse[r + 1]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < FIN_KEYS; ++k) {
    const int j = j0 + k * FIN_THREADS;
    at[k] = 0;
    if (page[k] >= a.n_pages) page[k] = -1;
    if (page[k] >= 0) {
      at[k] = ((size_t)page[k] * a.nkv + kvh) * a.page_size + j % a.page_size;
      if (j < old) sum[k] += a.scores[at[k]];
    }
  }
#pragma unroll
  for (int k = 0; k < FIN_KEYS; ++k) {
    const int j = j0 + k * FIN_THREADS;
    if (page[k] < 0) continue;
    a.scores_out[at[k]] = sum[k];
    if (j >= old && a.births) a.births[at[k]] = a.positions[first + j - old];
  }
}

inline cudaError_t launch_blocks(void (*kernel)(ShortArgs), dim3 grid, size_t smem, cudaStream_t stream, const ShortArgs& w) {
  return w.cluster ? nhv_launch_cluster(kernel, grid, SH_THREADS, smem, stream, w.cluster, w) : nhv_launch(kernel, grid, SH_THREADS, smem, stream, w);
}

template <int DB, int NT>
int launch_split(const ShortArgs& w, dim3 grid, size_t smem, cudaStream_t stream) {
  static std::atomic<uint64_t> done16{0}, done{0};
  if (w.a.page_size % 16 == 0) {
    NHV_CUDA(nhv_allow_smem((const void*)scored_short_kernel<DB, NT, true>, SH_MOST_SMEM, done16), "scored attention");
    NHV_CUDA(launch_blocks(scored_short_kernel<DB, NT, true>, grid, smem, stream, w), "scored attention");
  } else {
    NHV_CUDA(nhv_allow_smem((const void*)scored_short_kernel<DB, NT, false>, SH_MOST_SMEM, done), "scored attention");
    NHV_CUDA(launch_blocks(scored_short_kernel<DB, NT, false>, grid, smem, stream, w), "scored attention");
  }
  return 0;
}

template <int LPK, int EV, int RB>
int launch_f32(const ShortArgs& w, dim3 grid, size_t smem, cudaStream_t stream) {
  constexpr int BATCH = (RB * EV >= 32 ? 4 : 8) * 32 / LPK;
  static std::atomic<uint64_t> done{0}, done_by_page{0};
  if (w.a.page_size % BATCH == 0) {
    NHV_CUDA(nhv_allow_smem((const void*)scored_short_f32_kernel<LPK, EV, RB, true>, SH_MOST_SMEM, done_by_page), "scored attention");
    NHV_CUDA(launch_blocks(scored_short_f32_kernel<LPK, EV, RB, true>, grid, smem, stream, w), "scored attention");
  } else {
    NHV_CUDA(nhv_allow_smem((const void*)scored_short_f32_kernel<LPK, EV, RB, false>, SH_MOST_SMEM, done), "scored attention");
    NHV_CUDA(launch_blocks(scored_short_f32_kernel<LPK, EV, RB, false>, grid, smem, stream, w), "scored attention");
  }
  return 0;
}
template <int LPK, int EV>
int launch_f32(const ShortArgs& w, dim3 grid, size_t smem, cudaStream_t stream) {
  return w.block_rows <= 2 ? launch_f32<LPK, EV, 2>(w, grid, smem, stream) : w.block_rows <= 4 ? launch_f32<LPK, EV, 4>(w, grid, smem, stream)
                                                                                                : launch_f32<LPK, EV, 8>(w, grid, smem, stream);
}

}  // namespace

int scored_short_rows(int dtype, int d) {
  // float32: as many as the arrays of the second kernel hold.  Against the tiles of scored_attention.cu, 8 requests of 2,000 keys, 8 KV heads
  // of 128: 24 rows 155 us and 247, 32 rows 199 and 277; heads of 256 319 and 729; the tiles win only for 64 requests of 300 keys with heads
  // of 64 (179 and 171).
  // bfloat16: against the tcgen05 kernels, heads of 128, 24 rows: 2 requests of 20,000 keys 87 us and 96, 64 of 2,000 keys 255 and 291, 64 of
  // 300 107 and 96, 8 of 2,000 63 and 47; 32 rows: 112 and 96, 375 and 291, 138 and 96, 75 and 47.  Heads of 64, 32 rows: 81 and 81, 229
  // and 315, 89 and 86, 54 and 44.  A block's 16 rows of heads above 128 would need more registers than a thread has.
  return dtype == NHV_F32 ? 32 : d <= 64 ? 32 : d <= 128 ? 24 : 8;
}

bool scored_short_takes(int dtype, int rows, int d) {
  return d % (dtype == NHV_F32 ? 4 : 8) == 0 && d <= SA_MAX_D && rows <= scored_short_rows(dtype, d);
}

ShortPlan scored_short_plan(int dtype, int n_seqs, int max_rows, int max_keys, int nkv, int d) {
  ShortPlan p = {};
  p.rows = max_rows > 1 ? (max_rows + 1) / 2 * 2 : 2;      // requests that bring nothing go this way too: their scores pass through
  const int most = dtype == NHV_F32 ? 8 : 24;
  p.row_blocks = (p.rows + most - 1) / most;
  p.block_rows = (p.rows / p.row_blocks + (p.rows % p.row_blocks ? 1 : 0) + 1) / 2 * 2;
  // Four times as many blocks as run at once (three times took 4 and 2 % longer for drafts and 64 decoded tokens), so that requests of
  // unlike length even out, and no fewer than 64 keys a block (a tile per warp).
  const int an_sm = dtype == NHV_F32 ? (d <= 128 ? 3 : 2) : p.block_rows * ((d + 63) / 64) <= 16 ? 3 : 2, at_once = 148 * an_sm;
  const long long keys = (long long)n_seqs * nkv * p.row_blocks * max_keys, want = (keys + 4 * at_once - 1) / (4 * at_once);
  p.split_keys = (int)((want + 63) / 64 * 64);
  if (p.split_keys < 64) p.split_keys = 64;
  p.splits = (max_keys + p.split_keys - 1) / p.split_keys;
  // Where a request's parts are few, their scores stay in shared memory and all blocks run at once, a cluster of blocks
  // finishes the request and KV head alone, without a second launch: one request of 517 keys 18.4 -> 15.3 us a call, as long on the
  // device (9.8 against 9.5; float32 13.1 against 11.3), four of 1,000 keys 14.6 -> 11.6 there (float32 19.6 -> 16.3).  With more
  // blocks than that the wait for the slowest of a cluster costs more than the second kernel (64 requests 18 % longer).
  if (p.row_blocks == 1 && p.splits <= 2 * SH_MOST_CLUSTER) {
    int blocks = 1;
    while (blocks < p.splits && blocks < SH_MOST_CLUSTER) blocks *= 2;
    const int keys = (max_keys + blocks * 64 - 1) / (blocks * 64) * 64;
    const size_t smem = sizeof(float) * (short_sums(p.block_rows, d) + short_part(p.block_rows, d) + (size_t)keys * p.rows);
    if (smem <= 72 * 1024 && (long long)n_seqs * nkv * blocks <= at_once) {
      p.cluster = p.splits = blocks;
      p.split_keys = keys;
      p.smem = smem;
      p.group = n_seqs;
      return p;
    }
  }
  p.smem = sizeof(float) * short_sums(p.block_rows, d);
  p.keys = ((size_t)max_keys + 63) / 64 * 64;
  const size_t per_request = (size_t)nkv * p.rows * (p.keys + (size_t)p.splits * (d + 2));
  p.group = (int)(SH_MOST_SCORES / per_request);
  if (p.group < 1) p.group = 1;
  if (p.group > n_seqs) p.group = n_seqs;
  p.floats = per_request * p.group;
  return p;
}

// A request has at most 4 blocks that run at once / (requests x KV heads) parts and one that is not full.
size_t scored_short_most(int dtype, int n_seqs, int max_keys, int G, int nkv, int d) {
  const int rows = scored_short_rows(dtype, d);
  if (!scored_short_takes(dtype, G, d)) return 0;
  auto sum = [&](size_t n) { return n * nkv * rows * (((size_t)max_keys + 63) / 64 * 64) + (4 * 3 * 148 + n * nkv) * rows * (d + 2); };
  const size_t one = sum(1) > SH_MOST_SCORES ? sum(1) : SH_MOST_SCORES, all = sum(n_seqs);
  return all < one ? all : one;
}

int scored_short_launch(int dtype, ScoredArgs a, const ShortPlan& plan, float* work, cudaStream_t stream) {
  ShortArgs w = {};
  w.a = a;
  w.cap = nhv_score_cap(a.scale, a.softcap);
  w.keys = plan.keys;
  w.rows = plan.rows;
  w.block_rows = plan.block_rows;
  w.row_blocks = plan.row_blocks;
  w.split_keys = plan.split_keys;
  w.splits = plan.splits;
  w.cluster = plan.cluster;
  const size_t pairs = (size_t)plan.group * a.nkv;
  w.kept = work;
  w.part_o = w.kept + pairs * plan.keys * plan.rows;
  w.part_ml = w.part_o + pairs * plan.splits * plan.rows * a.d;
  const int db = (a.d + 63) / 64;
  const size_t smem = plan.smem;
  const int per_block = FIN_KEYS * FIN_THREADS;
  const int key_blocks = (a.max_keys + per_block - 1) / per_block, out_blocks = (plan.rows * a.d + FIN_THREADS - 1) / FIN_THREADS;
  for (int s = 0; s < a.n_seqs; s += plan.group) {
    w.first_seq = s;
    const int count = a.n_seqs - s < plan.group ? a.n_seqs - s : plan.group;
    const dim3 grid(plan.splits * plan.row_blocks, a.nkv, count);
    int rc = 0;
    if (dtype == NHV_F32)
      rc = a.d <= 32 ? launch_f32<8, 4>(w, grid, smem, stream) : a.d <= 64 ? launch_f32<16, 4>(w, grid, smem, stream)
           : a.d <= 128 ? launch_f32<32, 4>(w, grid, smem, stream) : launch_f32<32, 8>(w, grid, smem, stream);
    else if (plan.block_rows <= 8)
      rc = db == 1 ? launch_split<1, 1>(w, grid, smem, stream) : db == 2 ? launch_split<2, 1>(w, grid, smem, stream)
           : db == 3 ? launch_split<3, 1>(w, grid, smem, stream) : launch_split<4, 1>(w, grid, smem, stream);
    else if (plan.block_rows <= 16)
      rc = db == 1 ? launch_split<1, 2>(w, grid, smem, stream) : launch_split<2, 2>(w, grid, smem, stream);
    else
      rc = db == 1 ? launch_split<1, 3>(w, grid, smem, stream) : launch_split<2, 3>(w, grid, smem, stream);
    if (rc) return rc;
    if (w.cluster) return 0;                      // one group
    const dim3 all(key_blocks + out_blocks, a.nkv, count);
    if (dtype == NHV_F32) NHV_CUDA(nhv_launch(scored_short_finish_kernel<float>, all, FIN_THREADS, 0, stream, w, key_blocks, per_block), "scored attention");
    else NHV_CUDA(nhv_launch(scored_short_finish_kernel<__nv_bfloat16>, all, FIN_THREADS, 0, stream, w, key_blocks, per_block), "scored attention");
  }
  return 0;
}
