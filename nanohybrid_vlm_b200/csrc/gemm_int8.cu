// out[t, n] = (sum_k x[t, k] w[n, k]) * x_scales[t] * w_scales[n] for x [T, K] and w [N, K] of 8-bit integers; out bfloat16 or float32.
//
// The sum is exact in 32 bits (K <= 131,071: K * 128 * 128 < 2^31), so no cut of K and no order of adding changes an output: only the
// conversion of the sum to a float and the products with the two scales round (24 bits each), and the store once more.
//
// Two families on the tensor cores of the 5th generation, tcgen05.mma kind::i8 with 32-bit sums in tensor memory and both operands by TMA
// (128-byte swizzle; what lies behind a matrix arrives as zeros, so no size needs padding):
//   up to 128 tokens, where the weight's one read is the work: product_split_kernel, rows of the weight on the MMA's M axis;
//   more, where the arithmetic is: product_pair_kernel, pairs of SMs on tiles of 256 tokens.
// B200: 8 x 4,096 x 24,576 18 us (5.5 TB/s of weight; reading it alone takes 16.5), 64 x 12,288 x 4,096 13.2, 2,048 x 4,096 x 24,576 116 us in a prompt's step
// (3.55 POP/s; back to back for a while the power cap leaves 2.7 to 3.2).
#include <limits.h>
#include <string.h>

#ifndef NHV_WAIT_LIMIT
#define NHV_WAIT_LIMIT (1u << 22)
#endif
#include "nhv_async.cuh"
#include "nhv_overlap.h"

// Test builds only (tests compile this file into a library of its own with a short NHV_WAIT_LIMIT): the producers leave stage
// NHV_TEST_DROP_UNIT unsent, so that the waits for it run out.
#ifdef NHV_TEST_DROP_UNIT
#define NHV_UNIT_IS_SENT(i) ((i) != (NHV_TEST_DROP_UNIT))
#else
#define NHV_UNIT_IS_SENT(i) true
#endif

namespace {

typedef __nv_bfloat16 bf16;

struct Product {
  const int8_t *x, *w;
  const float *x_scales, *w_scales;
  void* out;
  long long x_stride, w_stride, out_stride;
  int T, N, K, out_f32;
  int boxes;             // rows of out start and end at multiples of 16 bytes
};

__device__ __forceinline__ float scaled(int sum, float xs, float ws) { return (float)sum * xs * ws; }

__device__ __forceinline__ void store_out(const Product& p, int t, int n, float v) {
  const long long at = (long long)t * p.out_stride + n;
  if (p.out_f32)
    reinterpret_cast<float*>(p.out)[at] = v;
  else
    reinterpret_cast<bf16*>(p.out)[at] = __float2bfloat16_rn(v);
}

// ---------------------------------------------------------------- rows that start anywhere
// Laid out anew with rows at multiples of 16 bytes, which all products read: a thread's 16 bytes of the copy come from the words that hold
// them, and no word is read that holds none of the row's.
__global__ void __launch_bounds__(256) align_rows_kernel(uint4* __restrict__ out, const int8_t* __restrict__ in, long long stride, long long pieces, int per_row,
                                                         int K) {
  pdl_prologue();
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= pieces) return;
  const long long row = i / per_row;
  const int k = (int)(i - row * per_row) * 16;
  const uintptr_t from = (uintptr_t)in + row * stride + k, end = from + min(16, K - k);
  const uint32_t shift = (uint32_t)(from & 3) * 8;
  uint32_t w[5];
#pragma unroll
  for (int j = 0; j < 5; ++j) {
    const uintptr_t at = (from & ~(uintptr_t)3) + 4 * j;
    w[j] = at < end ? *reinterpret_cast<const uint32_t*>(at) : 0u;
  }
  out[i] = make_uint4(__funnelshift_r(w[0], w[1], shift), __funnelshift_r(w[1], w[2], shift), __funnelshift_r(w[2], w[3], shift),
                      __funnelshift_r(w[3], w[4], shift));
}

int align_rows(const int8_t** rows, long long* stride, void* copy, int n, int K, cudaStream_t stream) {
  if (((uintptr_t)*rows | (uintptr_t)*stride) % 16 == 0) return 0;
  NHV_REQUIRE(copy && (uintptr_t)copy % 16 == 0, "linear_int8: rows that start between multiples of 16 bytes come with room for a copy");
  const int per_row = (K + 15) / 16;
  const long long pieces = (long long)n * per_row, blocks = (pieces + 255) / 256;
  NHV_REQUIRE(blocks < (1LL << 31), "linear_int8: too many rows");
  NHV_CUDA(nhv_launch(align_rows_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, (uint4*)copy, *rows, *stride, pieces, per_row, K), "linear_int8");
  *rows = (const int8_t*)copy;
  *stride = (long long)per_row * 16;
  return 0;
}

// ---------------------------------------------------------------- tcgen05 (8-bit integers, 32-bit sums in tensor memory)
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// The address of a shared variable in another block of the cluster.
__device__ __forceinline__ uint32_t in_block(uint32_t mine, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(mine), "r"(rank));
  return a;
}
__device__ __forceinline__ void store_cluster4(uint32_t at, int a, int b, int c, int d) {
  asm volatile("st.shared::cluster.v4.s32 [%0], {%1, %2, %3, %4};\n" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
// One lane of a converged warp: MMAs are issued under this, their operands the same in every lane, so that they lie in uniform
// registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ uint32_t same_in_all(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
template <int GROUP>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t columns) {
  if (GROUP == 1)
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n"
                 "tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::"r"(smem_u32(slot)), "r"(columns) : "memory");
  else
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n"
                 "tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::"r"(smem_u32(slot)), "r"(columns) : "memory");
}
template <int GROUP>
__device__ __forceinline__ void tmem_dealloc(uint32_t at, uint32_t columns) {
  if (GROUP == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(at), "r"(columns) : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(at), "r"(columns) : "memory");
}
// The MMAs issued so far arrive on `bar` when they have completed; of a pair's, on the barrier at this place in both blocks.
template <int GROUP>
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  if (GROUP == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar)) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n"
                 ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
// D[tmem] (+)= A[smem] * B[smem]^T over 32 columns of K
template <int GROUP>
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (GROUP == 1)
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_ld16(int (&r)[16], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_ld32(int (&r)[32], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }

// Descriptor of a K-major operand tile in shared memory in the 128-byte swizzle: rows of 128 bytes, groups of 8 rows 1,024 bytes
// apart, the tile on a 1,024-byte boundary; 32, 64 or 96 bytes further for the other slices of 32 columns.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// Instruction descriptor: signed 8-bit integers, both K-major, 32-bit sums, M x N.
__device__ __forceinline__ uint32_t instr_desc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// A box of a tensor map asked into L2.  Where other kernels still write there this reads nothing that is used: L2 is where all copies
// meet.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];\n" ::"l"((uint64_t)map), "r"(x), "r"(y) : "memory");
}
// A box into this block's shared memory, counted on a barrier of either block of the pair.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n"
               ::"r"(smem_u32(dst)), "l"((uint64_t)map), "r"(x), "r"(y), "r"(bar) : "memory");
}

constexpr int BK = 128;                // columns of K per stage: one 128-byte swizzle row
constexpr int UMMA_K = 32;

struct alignas(64) Mapped {
  CUtensorMap w_map, x_map, out_map;
  Product p;
  int nt;             // tokens of a tile: the boxes of x_map, a multiple of 16
  int tiles_t, tiles_n, group;
  int rows, stages, w_bytes, ring_bytes;      // few tokens: rows of the weight of a tile, and the ring
  int share, parts_bytes;                     // tokens that a block of a cluster finishes, and room for all parts of theirs
};

// ---- up to 128 tokens: up to 128 rows of the weight on the MMA's M axis, the tokens on its N axis.
//
// A block takes a tile of the weight's rows and one part of K; the blocks of a tile are a cluster.  The tile's height is free: the TMA box has
// that many rows, the MMA reads 128 from the stage's start and the sums of the rows behind are not looked at.  So the weight's rows divide
// evenly over the SMs, whatever N is.  Warp roles: TMA producer, MMA issuer, eight epilogue warps.  Before it waits for the kernel before it the
// producer asks its first stages into L2 (not into shared memory: the weight may be that kernel's output).
//
// With K in parts every block sends each token's sums to the one of the cluster that finishes the token, 16 bytes a lane into the other's
// shared memory, and after one meeting that block adds them up, which is exact, and writes.  (Parked sums that the finisher reads
// from the others, with two meetings: 64 x 12,288 x 4,096 13.6 us against 12.7, 64 x 4,096 x 4,096 8.7 against 7.2.)
//
// What bounds it: memory while a block streams (two blocks an SM, some 200 KB on their way); start and end of a launch, 3 us, beside that; with
// 64 tokens and more also what the tiles read of x, from L2.  The MMA issuer's operands are the same in every lane and the compiler has to see
// that (the warp's number by a shuffle, elect.sync): 407 -> 305 cycles a stage.
constexpr int SPLIT_THREADS = 320;     // producer warp, MMA warp, eight epilogue warps

// One output of each of up to 16 tokens.
template <typename O>
__device__ __forceinline__ void store_column16(O* at, long long stride, const int (&v)[16], const float* xs, float ws, int tokens) {
  if (tokens >= 16) {
#pragma unroll
    for (int j = 0; j < 16; ++j) at[j * stride] = from_f32<O>(scaled(v[j], xs[j], ws));
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < tokens) at[j * stride] = from_f32<O>(scaled(v[j], xs[j], ws));
  }
}
__global__ void __launch_bounds__(SPLIT_THREADS) product_split_kernel(const __grid_constant__ Mapped m) {
  const int STAGES = m.stages, W_BYTES = m.w_bytes, STAGE_BYTES = W_BYTES + m.nt * BK;
  const uint32_t COLUMNS = m.nt <= 32 ? 32 : m.nt <= 64 ? 64 : 128;
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* ring = smem_unaligned + ((1024 - (smem_u32(smem_unaligned) & 1023)) & 1023);
  int* parts = reinterpret_cast<int*>(ring + m.ring_bytes);       // [part][share of the tokens / 4][128][4]
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + m.ring_bytes + m.parts_bytes);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  __shared__ int s_abort;
  __shared__ float s_xs[128];

  const Product& p = m.p;
  const int warp = (int)same_in_all(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int S = m.group, rank = S > 1 ? (int)cluster_rank() : 0;
  const int n0 = (int)(blockIdx.x / S) * m.rows, n_end = min(n0 + m.rows, p.N), t0 = (int)blockIdx.y * m.nt;
  const int tokens = min(m.nt, p.T - t0);
  const int kt = (p.K + BK - 1) / BK;
  const int k0 = (int)((long long)kt * rank / S), k1 = (int)((long long)kt * (rank + 1) / S);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 1) tmem_alloc<1>(tmem_slot, COLUMNS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = same_in_all(*tmem_slot);
  pdl_launch_dependents();
  if (S > 1) cluster_arrive();

  if (warp == 0) {
    if (elect_one()) {
      const int n = k1 - k0;
      asm volatile("prefetch.tensormap [%0];\n" ::"l"((uint64_t)&m.x_map) : "memory");
      for (int i = 0; i < min(n, STAGES); ++i) tma_prefetch_2d(&m.w_map, (k0 + i) * BK, n0);
      pdl_wait();
      const uint32_t bytes = (m.rows + m.nt) * BK;                // zero-filled parts of a box count too
      uint32_t s = 0, phase = 1;
      for (int i = 0; i < n; ++i) {
        if (i >= STAGES && !mbar_wait(&empty[s], phase, 1)) { s_abort = 1; break; }
        if (NHV_UNIT_IS_SENT(i)) {
          unsigned char* dst = ring + (size_t)s * STAGE_BYTES;
          mbar_expect_tx(&full[s], bytes);
          tma_load_2d(dst, &m.w_map, (k0 + i) * BK, n0, &full[s]);
          tma_load_2d(dst + W_BYTES, &m.x_map, (k0 + i) * BK, t0, &full[s]);
        }
        if (++s == (uint32_t)STAGES) { s = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    pdl_wait();                                                    // the waits' limit counts from here, however long the kernel before takes
    const uint32_t idesc = instr_desc(128, m.nt);
    const int n = (int)same_in_all(k1 - k0);
    bool ok = true;
    uint32_t s = 0, phase = 0;
    const uint64_t first = smem_desc(same_in_all(smem_u32(ring)));
    for (int i = 0; i < n; ++i) {
      ok = __all_sync(0xffffffffu, mbar_wait(&full[s], phase, 2));
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t a = first + (uint64_t)(s * (uint32_t)(STAGE_BYTES >> 4)), b = a + (uint32_t)(W_BYTES >> 4);
#pragma unroll
        for (int kk = 0; kk < BK / UMMA_K; ++kk)
          tc_mma<1>(tmem_base, a + kk * (UMMA_K >> 4), b + kk * (UMMA_K >> 4), idesc, (i > 0 || kk > 0) ? 1u : 0u);
        tc_commit<1>(&empty[s]);
        if (i == n - 1) tc_commit<1>(acc_full);
      }
      __syncwarp();
      if (++s == (uint32_t)STAGES) { s = 0; phase ^= 1; }
    }
    if (!ok) s_abort = 1;
  }
  if (warp >= 2) {
    const int tid = (int)threadIdx.x - 64;                       // 0 .. 255
    pdl_wait();
    if (tid < tokens) s_xs[tid] = p.x_scales[t0 + tid];
    asm volatile("bar.sync 1, 256;\n" ::: "memory");
    // the tensor-memory lanes that this warp may read; every second piece of 16 tokens is its
    const int quarter = warp & 3, row = quarter * 32 + lane, second = warp >= 6, n = n0 + row;
    const float ws = n < n_end ? p.w_scales[n] : 0.f;
    const bool ok = __all_sync(0xffffffffu, mbar_wait(acc_full, 0, 3));
    tc_fence_after();
    if (S > 1) cluster_wait();                                   // all blocks of the cluster run
    if (!ok) {
      s_abort = 1;
    } else {
      const uint32_t at = tmem_base + ((uint32_t)(quarter * 32) << 16);
      for (int c = second * 16; c < tokens; c += 32) {
        int v[16];
        tmem_ld16(v, at + c);
        tmem_ld_wait();
        if (S > 1) {                                             // four tokens' sums at a time to the block that finishes them
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            if (c + j >= tokens) break;
            const int owner = (c + j) / m.share, four = (c + j - owner * m.share) >> 2;
            const int* to = parts + (((rank * (m.share >> 2) + four) * 128 + row) << 2);
            store_cluster4(in_block(smem_u32(to), owner), v[j], v[j + 1], v[j + 2], v[j + 3]);
          }
        } else if (n < n_end) {
          const long long o = (long long)(t0 + c) * p.out_stride + n;
          if (p.out_f32)
            store_column16(reinterpret_cast<float*>(p.out) + o, p.out_stride, v, s_xs + c, ws, tokens - c);
          else
            store_column16(reinterpret_cast<bf16*>(p.out) + o, p.out_stride, v, s_xs + c, ws, tokens - c);
        }
      }
    }
    tc_fence_before();
    if (S > 1) {
      __syncwarp();
      cluster_arrive();
      cluster_wait();                                            // all parts have arrived
      const int j0 = rank * m.share, fours = (min(tokens, j0 + m.share) - j0 + 3) >> 2;
      for (int f = second; f < fours && n < n_end; f += 2) {
        const int4* from = reinterpret_cast<const int4*>(parts) + f * 128 + row;
        int4 part[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) part[q] = q < S ? from[q * (m.share >> 2) * 128] : make_int4(0, 0, 0, 0);
        int sum[4] = {};
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          sum[0] += part[q].x; sum[1] += part[q].y; sum[2] += part[q].z; sum[3] += part[q].w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + f * 4 + e;
          if (j < tokens) store_out(p, t0 + j, n, scaled(sum[e], s_xs[j], ws));
        }
      }
    }
  } else if (S > 1) {
    __syncwarp();
    cluster_wait();
    cluster_arrive();
    cluster_wait();
  }
  __syncthreads();
  if (s_abort) give_up_delay();                                  // let copies that may still be in flight land
  tc_fence_after();
  if (warp == 1) tmem_dealloc<1>(tmem_base, COLUMNS);
}

// ---- more than 128 tokens: pairs of blocks (cta_group::2), 256 tokens on the MMA's M axis (128 a block), TN outputs on its N axis (TN / 2 rows of
// the weight in each block's shared memory), tiles handed out in turn to a grid of one pair for two SMs.
//
// Bound by the tensor pipe (90 % of its cycles at 2,048 x 4,096 x 24,576) and, back to back, by the power cap.  A pair reads each operand's
// bytes once for both SMs, two accumulators let a tile's MMAs run beside the last one's epilogue, and outputs leave by TMA stores from 2 KB a
// warp (8,192 x 256 x 4,096 in bfloat16 25.8 -> 22.7 us, in float32 55 -> 40).  Block 0's barriers count both blocks' copies, commits reach both.
constexpr int PAIR_THREADS = 320;      // producer warp, MMA warp, eight epilogue warps
constexpr int TURN = 2560;             // bytes of a warp's outputs on their way out: 32 rows of 64 bytes, or of 17 floats; whole 512s for the swizzle
template <int TN>
struct Pair {
  static constexpr int X_BYTES = 128 * BK, W_BYTES = TN / 2 * BK, STAGE = X_BYTES + W_BYTES;      // a block's half of a stage
  static constexpr int STAGES = 196608 / STAGE;
  static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE + 8 * (TN / 2) * 4 + 8 * TURN + (2 * STAGES + 4) * 8 + 16;
};

// A warp's 32 outputs of 32 rows from (t0, n0): 64 bytes of each row at a time through 2 KB of shared memory in the 64-byte swizzle, from where
// a TMA store takes them while the warp goes on; what lies behind out's rows and columns is not written.  A row ends at a multiple of 16 bytes
// (Product::boxes): a store writes whole 16 bytes, with zeros behind the last column.
__device__ __forceinline__ void store_box(const CUtensorMap* map, unsigned char* box, const uint32_t (&w)[16], int n, int t, int lane) {
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");      // the last one has read the box
  __syncwarp();
  const uint32_t at = smem_u32(box) + lane * 64, turn = (lane >> 1) & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(at + ((i ^ turn) << 4)), "r"(w[4 * i]), "r"(w[4 * i + 1]), "r"(w[4 * i + 2]),
                 "r"(w[4 * i + 3]) : "memory");
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  __syncwarp();
  if (lane == 0)
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n"
                 "cp.async.bulk.commit_group;\n" ::"l"((uint64_t)map), "r"(n), "r"(t), "r"(smem_u32(box)) : "memory");
}
__device__ __forceinline__ void store_rows32(const CUtensorMap* map, unsigned char* box, const float (&v)[32], bool f32, int n0, int t0, int lane) {
  uint32_t w[16];
  if (f32) {
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[h + i]);
      store_box(map, box, w, n0 + h, t0, lane);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    store_box(map, box, w, n0, t0, lane);
  }
}
// The same where rows start or end at odd places: 16 columns of two rows at a time, lanes side by side.
template <typename O>
__device__ __forceinline__ void store_turned(O* out, const Product& p, float* mine, const float (&v)[32], int t0, int n0, int lane) {
#pragma unroll
  for (int h = 0; h < 32; h += 16) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; ++j) mine[lane * 17 + j] = v[h + j];
    __syncwarp();
    const int n = n0 + h + (lane & 15), t = t0 + (lane >> 4), rows = n < p.N ? p.T - t : 0;
    O* at = out + (long long)t * p.out_stride + n;
#pragma unroll
    for (int r = 0; r < 32; r += 2)
      if (r < rows) at[r * p.out_stride] = from_f32<O>(mine[(r + (lane >> 4)) * 17 + (lane & 15)]);
  }
  __syncwarp();
}

// The tile'th tile: `group` tiles of tokens after one another beside the same rows of the weight, then the next rows.
__device__ __forceinline__ void tile_place(const Mapped& m, int tile, int& tt, int& tn) {
  const int per = m.group * m.tiles_n, g = tile / per, r = tile - g * per;
  const int here = min(m.group, m.tiles_t - g * m.group);
  tn = r / here;
  tt = g * m.group + (r - tn * here);
}

template <int TN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1) product_pair_kernel(const __grid_constant__ Mapped m) {
  constexpr int STAGES = Pair<TN>::STAGES, STAGE = Pair<TN>::STAGE, X_BYTES = Pair<TN>::X_BYTES, HALF = TN / 2;
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* ring = smem_unaligned + ((1024 - (smem_u32(smem_unaligned) & 1023)) & 1023);
  unsigned char* boxes = ring + (size_t)STAGES * STAGE;                // [8 warps][TURN]
  float* scales = reinterpret_cast<float*>(boxes + 8 * TURN);      // [8 warps][HALF]
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + 8 * HALF);        // used in block 0, for both
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;      // [2]
  uint64_t* acc_empty = acc_full + 2;            // [2], used in block 0
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  __shared__ int s_abort;

  const Product& p = m.p;
  const int warp = (int)same_in_all(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pairs = gridDim.x >> 1, pair = blockIdx.x >> 1;
  const int tiles = m.tiles_t * m.tiles_n, kt = (p.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 16);              // eight warps of both blocks
    }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 1) tmem_alloc<2>(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();                                                // both blocks' barriers are there
  tc_fence_after();
  const uint32_t tmem_base = same_in_all(*tmem_slot);
  pdl_launch_dependents();
  pdl_wait();

  if (warp == 0) {
    if (elect_one()) {
      int i = 0;
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs) {
        int tt, tn;
        tile_place(m, tile, tt, tn);
        const int t0 = tt * 256 + (int)rank * 128, n0 = tn * TN + (int)rank * HALF;
        for (int k = 0; k < kt; ++k, ++i) {
          const int s = i % STAGES;
          if (i >= STAGES && !mbar_wait(&empty[s], (uint32_t)((i / STAGES) - 1) & 1, 1)) { ok = false; break; }
          if (!NHV_UNIT_IS_SENT(i)) continue;
          unsigned char* dst = ring + (size_t)s * STAGE;
          const uint32_t bar = in_block(smem_u32(&full[s]), 0);
          if (rank == 0) mbar_expect_tx(&full[s], 2 * STAGE);      // zero-filled parts of a box count too
          tma_load_2d_pair(dst, &m.x_map, k * BK, t0, bar);
          tma_load_2d_pair(dst + X_BYTES, &m.w_map, k * BK, n0, bar);
        }
      }
      // no block leaves before the last commits have reached it
      for (int j = max(0, i - STAGES); j < i && ok; ++j) ok = mbar_wait(&empty[j % STAGES], (uint32_t)(j / STAGES) & 1, 1);
      if (!ok) s_abort = 1;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc = instr_desc(256, TN);
      bool ok = true;
      int i = 0, turn = 0;
      for (int tile = pair; tile < tiles && ok; tile += pairs, ++turn) {
        if (turn >= 2) {
          ok = __all_sync(0xffffffffu, mbar_wait(&acc_empty[turn & 1], (uint32_t)((turn >> 1) - 1) & 1, 2));
          if (!ok) break;
          tc_fence_after();
        }
        const uint32_t d = tmem_base + (uint32_t)((turn & 1) * 256);
        for (int k = 0; k < kt; ++k, ++i) {
          const int s = i % STAGES;
          ok = __all_sync(0xffffffffu, mbar_wait(&full[s], (uint32_t)(i / STAGES) & 1, 3));
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t a = smem_desc(smem_u32(ring) + s * STAGE), b = a + (X_BYTES >> 4);
#pragma unroll
            for (int kk = 0; kk < BK / UMMA_K; ++kk)
              tc_mma<2>(d, a + kk * (UMMA_K >> 4), b + kk * (UMMA_K >> 4), idesc, (k > 0 || kk > 0) ? 1u : 0u);
            tc_commit<2>(&empty[s]);
            if (k == kt - 1) tc_commit<2>(&acc_full[turn & 1]);
          }
          __syncwarp();
        }
      }
      if (!ok) s_abort = 1;
    }
  } else {
    const int quarter = warp & 3, half = warp >= 6 ? HALF : 0;      // lanes that this warp may read; its columns
    float* mine = scales + (warp - 2) * HALF;
    int turn = 0;
    bool ok = true;
    for (int tile = pair; tile < tiles; tile += pairs, ++turn) {
      int tt, tn;
      tile_place(m, tile, tt, tn);
      const int t = tt * 256 + (int)rank * 128 + quarter * 32 + lane, n0 = tn * TN + half;
      const float xs = t < p.T ? p.x_scales[t] : 0.f;
#pragma unroll
      for (int j = 0; j < HALF / 32; ++j) {
        const int n = n0 + j * 32 + lane;
        mine[j * 32 + lane] = n < p.N ? p.w_scales[n] : 0.f;
      }
      __syncwarp();
      ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[turn & 1], (uint32_t)(turn >> 1) & 1, 4));
      if (!ok) break;
      tc_fence_after();
      const uint32_t at = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)((turn & 1) * 256 + half);
      for (int c = 0; c < HALF; c += 32) {
        int r[32];
        float v[32];
        tmem_ld32(r, at + c);
        tmem_ld_wait();
        if (c == HALF - 32) {                                             // the accumulator is read: the MMAs may have it again
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_cluster(in_block(smem_u32(&acc_empty[turn & 1]), 0));
        }
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 ws = *reinterpret_cast<const float4*>(mine + c + j);
          v[j] = scaled(r[j], xs, ws.x);
          v[j + 1] = scaled(r[j + 1], xs, ws.y);
          v[j + 2] = scaled(r[j + 2], xs, ws.z);
          v[j + 3] = scaled(r[j + 3], xs, ws.w);
        }
        if (n0 + c >= p.N || t - lane >= p.T) continue;
        unsigned char* box = boxes + (warp - 2) * TURN;
        if (p.boxes)
          store_rows32(&m.out_map, box, v, p.out_f32, n0 + c, t - lane, lane);
        else if (p.out_f32)
          store_turned(reinterpret_cast<float*>(p.out), p, reinterpret_cast<float*>(box), v, t - lane, n0 + c, lane);
        else
          store_turned(reinterpret_cast<bf16*>(p.out), p, reinterpret_cast<float*>(box), v, t - lane, n0 + c, lane);
      }
      __syncwarp();
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
    if (!ok) s_abort = 1;
  }
  __syncthreads();
  if (s_abort) give_up_delay();                                  // let copies that may still be in flight land
  cluster_sync();                                                // the other block's MMAs, commits and copies reach in here
  tc_fence_after();
  if (warp == 1) tmem_dealloc<2>(tmem_base, 512);
}

bool encode_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, long long rows, long long columns, long long stride_bytes, int box_columns,
                int box_rows, CUtensorMapSwizzle swizzle, CUtensorMapL2promotion promotion) {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = []() -> PFN_cuTensorMapEncodeTiled_v12000 {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess) return nullptr;
    return (PFN_cuTensorMapEncodeTiled_v12000)fn;
  }();
  if (!encode) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)columns, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride_bytes};
  const cuuint32_t box[2] = {(cuuint32_t)box_columns, (cuuint32_t)box_rows}, steps[2] = {1, 1};
  return encode(map, type, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, promotion,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Rows of bytes, read in boxes of 128 bytes x `box_rows` rows with the 128-byte swizzle.
bool make_map(CUtensorMap* map, const void* base, long long rows, long long bytes, long long stride, int box_rows) {
  return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, rows, bytes, stride, BK, box_rows, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}
// The output, written in boxes of 64 bytes x 32 rows with the 64-byte swizzle.
bool make_out_map(CUtensorMap* map, const Product& p) {
  const int item = p.out_f32 ? 4 : 2;
  return encode_map(map, p.out_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.out, p.T, p.N, p.out_stride * item, 64 / item, 32,
                    CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE);
}

struct SplitPlan {
  int nt, rows, parts, stages;
};

struct SplitSmem {
  int w_bytes, ring_bytes, share, parts_bytes;
  size_t all;
};
SplitSmem split_smem(const SplitPlan& plan) {
  SplitSmem s;
  s.w_bytes = (plan.rows * BK + 1023) / 1024 * 1024;
  // the MMAs read 128 rows from a stage's start, whatever lies there
  s.ring_bytes = (plan.stages - 1) * (s.w_bytes + plan.nt * BK) + 128 * BK + plan.nt * BK;
  s.share = ((plan.nt + plan.parts - 1) / plan.parts + 3) / 4 * 4;
  s.parts_bytes = plan.parts > 1 ? plan.parts * s.share * 512 : 0;
  s.all = 1024 + (size_t)s.ring_bytes + s.parts_bytes + (2 * plan.stages + 1) * 8 + 16;
  return s;
}

// Rows of a tile, parts of K and stages.  Times in us for 16 / 64 / 128 tokens.
//   K in one part, a tile for each SM or, where that would be more than 96 rows, two: 12,288 x 4,096: 84 rows 11.2 / 11.6 / 13.6, 42 rows
//   12.0 / 13.0 / 14.5; 24,576 x 4,096: 84 rows 18.8 / 19.1 / 22.0, 128 rows 19.9 / 20.5 / 23.4.  With a tile for each SM and more than 32 tokens the ring
//   takes most of the SM (10,240 x 4,096 - / 10.3 / 11.7, with half of it - / 10.8 / 13.9); else, and for short sums, half, so that the next kernel's
//   block finds room (9.8 against 10.1 with most; 10,240 x 1,024 4.5 / 5.2, with most - / 5.3).
//   Narrower weights: tiles of 128 rows, K over a cluster of blocks: 4,096 x 4,096 in 4 parts 5.7 / 7.1 / 9.3, in 1 with 28 rows 8.5 / 9.4 / 11.2;
//   10,240 x 4,096 in 3 9.6 / 12.2, 8,192 x 12,288 in 4 - / 21.6, in 1 - / 23.2, hence the bounds on N with more than 32 tokens.  Up to 64 tokens two
//   blocks share an SM (4,096 x 12,288 in 8 parts 11.0 / 13.2, in 4 11.8 / 13.0) unless a part would have fewer than 8 stages (4,096 x 4,096
//   in 8 parts: 6.3 / 8.2); above, the room for the parts' sums leaves a second block no ring.  A block alone on its SM has four stages at
//   least (4,096 x 4,096 with three - / 7.7).  Clusters that would fill the SMs to the last do not all find their places at once
//   (12,288 x 4,096 in 3 parts, 288 blocks: 15.1 / 19.6; 2,048 x 4,096 for 128 tokens as 16 clusters of 8 13.4, as 32 of 4 with tiles of 64 rows
//   8.6).
//   Short sums: K in one part, the tiles smaller: 4,096 x 1,024, 64 rows 3.6 / 4.1 / 5.1, 4 parts of 128 rows 3.6 / 5.3 / 8.8.
SplitPlan split_plan(int T, int N, int K, int sms) {
  const int kt = (K + BK - 1) / BK;
  SplitPlan plan;
  plan.nt = T >= 128 ? 128 : (T + 15) / 16 * 16;
  const bool shared = plan.nt <= 64, few = plan.nt <= 32;
  plan.rows = shared || N > 64 * (sms * 7 / 8 / 4) ? 128 : 64;
  int tiles = (N + plan.rows - 1) / plan.rows;
  const int most_parts = shared ? 8 : 4;
  plan.parts = (shared ? 2 * sms * 9 / 10 : sms * 7 / 8) / tiles;
  if (plan.parts > most_parts) plan.parts = most_parts;
  while (plan.parts > 1 && kt < 8 * plan.parts && tiles * plan.parts > sms) --plan.parts;
  if (plan.parts > kt) plan.parts = kt;
  if (plan.parts < (shared || kt < 32 ? 3 : 2) || (kt < 16 && N >= 24 * sms) || (!few && N >= (shared ? 60 : 48) * sms)) {
    plan.parts = 1;
    const long long slots = N > 96LL * sms ? 2 * sms : sms, waves = (N + 128LL * slots - 1) / (128LL * slots);
    plan.rows = (int)((N + waves * slots - 1) / (waves * slots));
    if (plan.rows < 32) plan.rows = N < 64 ? 64 : 32;
    tiles = (N + plan.rows - 1) / plan.rows;
  }
  const bool alone = !few && kt >= 16 && (long long)tiles * plan.parts <= sms;
  const size_t most = ((plan.parts == 1 ? alone : !shared) ? 200 : 112) * 1024;
  const int least = alone && plan.parts <= 4 ? 4 : 1;
  plan.stages = 8;
  while (plan.stages > least && split_smem(plan).all > most) --plan.stages;
  return plan;
}

int split_product(Mapped& m, const SplitPlan& plan, cudaStream_t stream) {
  const Product& p = m.p;
  NHV_REQUIRE(plan.rows >= 1 && plan.rows <= 128 && plan.nt >= 16 && plan.nt <= 128 && plan.nt % 16 == 0 && plan.stages >= 1 && plan.stages <= 16 && plan.parts >= 1 &&
              plan.parts <= 8, "linear_int8: tiles of %d rows and %d tokens, %d stages, %d parts", plan.rows, plan.nt, plan.stages, plan.parts);
  m.nt = plan.nt;
  m.rows = plan.rows;
  m.group = plan.parts;
  m.stages = plan.stages;
  m.tiles_t = (p.T + m.nt - 1) / m.nt;
  m.tiles_n = (p.N + m.rows - 1) / m.rows;
  const SplitSmem room = split_smem(plan);
  m.w_bytes = room.w_bytes;
  m.ring_bytes = room.ring_bytes;
  m.share = room.share;
  m.parts_bytes = room.parts_bytes;
  NHV_REQUIRE(room.all <= 225 * 1024, "linear_int8: a ring of %d bytes", m.ring_bytes);
  NHV_REQUIRE(make_map(&m.w_map, p.w, p.N, p.K, p.w_stride, m.rows) && make_map(&m.x_map, p.x, p.T, p.K, p.x_stride, m.nt),
              "linear_int8: cannot encode the tensor maps");
  static std::atomic<uint64_t> allowed{0};
  NHV_CUDA(nhv_allow_smem((const void*)product_split_kernel, 225 * 1024, allowed), "linear_int8");
  NHV_CUDA(nhv_launch_cluster(product_split_kernel, dim3(m.tiles_n * m.group, m.tiles_t), dim3(SPLIT_THREADS), room.all, stream, m.group, m),
           "linear_int8");
  return 0;
}

template <int TN>
int launch_pair(Mapped& m, int sms, cudaStream_t stream) {
  const Product& p = m.p;
  m.nt = 256;
  m.tiles_t = (p.T + 255) / 256;
  m.tiles_n = (p.N + TN - 1) / TN;
  m.group = m.tiles_t < 16 ? m.tiles_t : 16;
  NHV_REQUIRE(make_map(&m.w_map, p.w, p.N, p.K, p.w_stride, TN / 2) && make_map(&m.x_map, p.x, p.T, p.K, p.x_stride, 128) &&
              (!p.boxes || make_out_map(&m.out_map, p)), "linear_int8: cannot encode the tensor maps");
  const long long tiles = (long long)m.tiles_t * m.tiles_n;
  NHV_REQUIRE(tiles < (1LL << 30), "linear_int8: too many tiles");
  const int pairs = (int)(tiles < sms / 2 ? tiles : sms / 2);
  static std::atomic<uint64_t> allowed{0};
  NHV_CUDA(nhv_allow_smem((const void*)product_pair_kernel<TN>, (int)Pair<TN>::SMEM, allowed), "linear_int8");
  NHV_CUDA(nhv_launch(product_pair_kernel<TN>, dim3(2 * pairs), dim3(PAIR_THREADS), Pair<TN>::SMEM, stream, m), "linear_int8");
  return 0;
}

// The tiles' width: the one with the least turns * (width + 64), a turn being a tile for every pair, and 64 what a tile costs beside
// its width.  us for widths 64 / 128 / 192 / 256: 256 tokens, 4,096 x 4,096 9.3 / 9.9 / - / 15.0, 24,576 x 4,096 35.5 / 26.5 / 26.2 / 29.0; 4,096 x 12,288, 512
// tokens 32.4 / 23.1 / 31.0 / 36.0, 1,024 - / 39.1 / 47.7 / 37.1, 2,048 - / 90.7 / 84.2 / 75.4.
struct PairPlan {
  int width;
  long long tiles, turns;
};
PairPlan pair_plan(int T, int N, int sms) {
  const long long tiles_t = (T + 255) / 256, pairs = sms / 2;
  PairPlan plan = {};
  for (int w = 256; w >= 64; w -= 64) {
    const long long tiles = tiles_t * ((N + w - 1) / w), turns = (tiles + pairs - 1) / pairs;
    if (w == 256 || turns * (w + 64) < plan.turns * (plan.width + 64)) plan = {w, tiles, turns};
  }
  return plan;
}

int pair_product(Mapped& m, int sms, cudaStream_t stream) {
  const int width = pair_plan(m.p.T, m.p.N, sms).width;
  if (width == 64) return launch_pair<64>(m, sms, stream);
  if (width == 128) return launch_pair<128>(m, sms, stream);
  if (width == 192) return launch_pair<192>(m, sms, stream);
  return launch_pair<256>(m, sms, stream);
}

}  // namespace

// Reads and clears the error word (0: no bounded wait ever ran out).  Synchronises the device.
NHV_API int nhv_gemm_int8_error() { return nhv_wait_error_take(); }
// The device address of the error word, for kernels that report it with the step's result.
NHV_API void* nhv_gemm_int8_error_word() { return nhv_wait_error_address(); }

// How a product of these sizes is cut on a device with `sms` SMs, in `out`: 0 (K may be in parts) or 1 (pairs of SMs), tokens of a tile, outputs of a
// tile, parts of K, stages of the ring, tiles, turns of a pair, bytes of shared memory of a block.
NHV_API int nhv_gemm_int8_plan(int T, int N, int K, int sms, long long* out) {
  NHV_REQUIRE(T > 0 && N > 0 && K > 0 && K <= 131071 && T <= INT_MAX - 511 && N <= INT_MAX - 511 && sms > 1 && out, "linear_int8: no plan for these sizes");
  if (T <= 128) {
    const SplitPlan plan = split_plan(T, N, K, sms);
    const long long all[8] = {0, plan.nt, plan.rows, plan.parts, plan.stages, (N + plan.rows - 1) / plan.rows, 1, (long long)split_smem(plan).all};
    memcpy(out, all, sizeof(all));
  } else {
    const PairPlan plan = pair_plan(T, N, sms);
    const int stages[4] = {Pair<64>::STAGES, Pair<128>::STAGES, Pair<192>::STAGES, Pair<256>::STAGES};
    const size_t smem[4] = {Pair<64>::SMEM, Pair<128>::SMEM, Pair<192>::SMEM, Pair<256>::SMEM};
    const int i = plan.width / 64 - 1;
    const long long all[8] = {1, 256, plan.width, 1, stages[i], plan.tiles, plan.turns, (long long)smem[i]};
    memcpy(out, all, sizeof(all));
  }
  return 0;
}

// What a call is given, one after the other, in one block.
struct ProductCall {
  long long out, x, x_scales, w, w_scales, x_copy, w_copy, out_stride, x_stride, w_stride;      // the copies: room for rows that start anywhere, or 0
  int out_dtype, T, N, K;
};

// The SMs of the current device, asked for once.
static int sm_count() {
  static std::atomic<int> known[64];
  int device = 0, n = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return 0;
  if (device < 64) n = known[device].load(std::memory_order_relaxed);
  if (n == 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) == cudaSuccess && device < 64)
    known[device].store(n, std::memory_order_relaxed);
  return n;
}

NHV_API int nhv_gemm_int8(const void* given, cudaStream_t stream) {
  ProductCall c;
  memcpy(&c, given, sizeof(c));
  const int T = c.T, N = c.N, K = c.K, sms = sm_count();
  if (T == 0 || N == 0) return 0;
  NHV_REQUIRE(T > 0 && N > 0 && K > 0 && K <= 131071, "linear_int8: a sum over 1 to 131,071 products is exact in 32 bits, not over %d", K);
  NHV_REQUIRE(T <= INT_MAX - 511 && N <= INT_MAX - 511, "linear_int8: %d tokens and %d outputs: a tile's last row has no number in 32 bits", T, N);
  NHV_REQUIRE(c.out && c.x && c.w && c.x_scales && c.w_scales && (c.out_dtype == NHV_F32 || c.out_dtype == NHV_BF16), "linear_int8: bad arguments");
  const long long item = c.out_dtype == NHV_F32 ? 4 : 2;
  const NhvRows out = {c.out, T, c.out_stride * item, N * item};
  NHV_REQUIRE(!nhv_rows_meet(out, {c.x, T, c.x_stride, K}) && !nhv_rows_meet(out, {c.w, N, c.w_stride, K}) &&
              !nhv_rows_meet(out, {c.x_scales, 1, 0, 4LL * T}) && !nhv_rows_meet(out, {c.w_scales, 1, 0, 4LL * N}),
              "the output has memory of its own: operands and scales are read again for other outputs");
  NHV_REQUIRE(sms > 1, "linear_int8: the device does not say how many SMs it has");
  Product p = {(const int8_t*)c.x, (const int8_t*)c.w, (const float*)c.x_scales, (const float*)c.w_scales, (void*)c.out,
                     c.x_stride, c.w_stride, c.out_stride, T, N, K, c.out_dtype == NHV_F32,
                     (c.out | c.out_stride * item | N * item) % 16 == 0};
  if (int e = align_rows(&p.x, &p.x_stride, (void*)c.x_copy, T, K, stream)) return e;
  if (int e = align_rows(&p.w, &p.w_stride, (void*)c.w_copy, N, K, stream)) return e;
  // us, whole tiles of the weight / pairs: 128 tokens, 4,096 x 4,096 9.4 / 9.3, 24,576 x 4,096 22.1 / 26.2, 4,096 x 12,288 14.9 / 18.6; 256 tokens 12.7 / 9.3,
  // 33 / 26.2, 19.5 / 18.6.  Up to 8 tokens the weight through registers into mma.sync was tried: alone 5.0, 18.5 and 10.6 against 6.0, 18.3 and 11.0,
  // but in a decode step, behind other kernels, 7.2, 31.5 and 18.3 against 5.1, 17.8 and 8.5 (its blocks fill an SM, so that none starts under
  // the kernel before).
  Mapped m;
  m.p = p;
  if (T <= 128) return split_product(m, split_plan(T, N, K, sms), stream);
  return pair_product(m, sms, stream);
}
