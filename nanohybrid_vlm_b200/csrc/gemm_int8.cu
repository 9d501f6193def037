// out[t, n] = (sum_k x[t, k] w[n, k]) * x_scales[t] * w_scales[n] for x [T, K] and w [N, K] of 8-bit integers; out bfloat16 or float32.
//
// The sum is exact in 32 bits (K <= 131,071: K * 128 * 128 < 2^31), so no cut of K and no order of adding changes an output: only the
// conversion of the sum to a float and the products with the two scales round, and the store once more.
#define NHV_WAIT_LIMIT (1u << 22)
#include "nhv_async.cuh"

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
__device__ __forceinline__ int4 load_cluster4(uint32_t at) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
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
  CUtensorMap w_map, x_map;
  Product p;
  int nt;             // tokens of a tile: the boxes of x_map, a multiple of 16
  int tiles_t, tiles_n, group;
};

// ---- few tokens: 128 rows of the weight on the MMA's M axis, up to NT tokens on its N axis.
constexpr int SPLIT_THREADS = 192;     // producer warp, MMA warp, four epilogue warps
constexpr int W_BYTES = 128 * BK;

template <int NT, int STAGES>
__global__ void __launch_bounds__(SPLIT_THREADS) product_split_kernel(const __grid_constant__ Mapped m) {
  constexpr int STAGE_BYTES = W_BYTES + NT * BK;
  constexpr uint32_t COLUMNS = NT < 32 ? 32 : NT;
  static_assert((size_t)STAGES * STAGE_BYTES >= (size_t)NT * 512, "the sums are parked over the ring");
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* ring = smem_unaligned + ((1024 - (smem_u32(smem_unaligned) & 1023)) & 1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + (size_t)STAGES * STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  __shared__ int s_abort;

  const Product& p = m.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = m.group, rank = S > 1 ? (int)cluster_rank() : 0;
  const int n0 = (int)(blockIdx.x / S) * 128, t0 = (int)blockIdx.y * m.nt;
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
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();

  if (warp == 0) {
    if (elect_one()) {
      const int n = k1 - k0;
      for (int i = 0; i < min(n, STAGES); ++i) tma_prefetch_2d(&m.w_map, (k0 + i) * BK, n0);
      pdl_wait();
      const uint32_t bytes = W_BYTES + m.nt * BK;                // zero-filled parts of a box count too
      for (int i = 0; i < n; ++i) {
        const int s = i % STAGES;
        if (i >= STAGES && !mbar_wait(&empty[s], (uint32_t)((i / STAGES) - 1) & 1, 1)) { s_abort = 1; break; }
        unsigned char* dst = ring + (size_t)s * STAGE_BYTES;
        mbar_expect_tx(&full[s], bytes);
        tma_load_2d(dst, &m.w_map, (k0 + i) * BK, n0, &full[s]);
        tma_load_2d(dst + W_BYTES, &m.x_map, (k0 + i) * BK, t0, &full[s]);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t idesc = instr_desc(128, m.nt);
    bool ok = true;
    for (int i = 0; i < k1 - k0; ++i) {
      const int s = i % STAGES;
      ok = __all_sync(0xffffffffu, mbar_wait(&full[s], (uint32_t)(i / STAGES) & 1, 2));
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t a = smem_desc(smem_u32(ring) + s * STAGE_BYTES), b = a + (W_BYTES >> 4);
#pragma unroll
        for (int kk = 0; kk < BK / UMMA_K; ++kk)
          tc_mma<1>(tmem_base, a + kk * (UMMA_K >> 4), b + kk * (UMMA_K >> 4), idesc, (i > 0 || kk > 0) ? 1u : 0u);
        tc_commit<1>(&empty[s]);
        if (i == k1 - k0 - 1) tc_commit<1>(acc_full);
      }
      __syncwarp();
    }
    if (!ok) s_abort = 1;
  }
  const int tid = (int)threadIdx.x - 64;                         // the epilogue's threads: 0 .. 127
  int* parked = reinterpret_cast<int*>(ring);                    // [token][128]
  if (warp >= 2) {
    pdl_wait();
    const int quarter = warp & 3, row = quarter * 32 + lane, n = n0 + row;      // the tensor-memory lanes that this warp may read
    const float ws = n < p.N ? p.w_scales[n] : 0.f;
    const bool ok = __all_sync(0xffffffffu, mbar_wait(acc_full, 0, 3));
    tc_fence_after();
    if (!ok) {
      s_abort = 1;
    } else {
      const uint32_t at = tmem_base + ((uint32_t)(quarter * 32) << 16);
      for (int c = 0; c < tokens; c += 16) {
        int v[16];
        tmem_ld16(v, at + c);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (S > 1)
            parked[(c + j) * 128 + row] = v[j];
          else if (c + j < tokens && n < p.N)
            store_out(p, t0 + c + j, n, scaled(v[j], p.x_scales[t0 + c + j], ws));
        }
      }
    }
    tc_fence_before();
  }
  if (S > 1) {
    __syncwarp();
    cluster_sync();                                              // every block's sums are parked
    if (warp >= 2) {
      const int items = tokens * 32;
      for (int i = items * rank / S + tid; i < items * (rank + 1) / S; i += 128) {
        const int j = i >> 5, n = n0 + 4 * (i & 31);
        const uint32_t mine = smem_u32(parked + i * 4);
        int4 sum = make_int4(0, 0, 0, 0);
        for (int q = 0; q < S; ++q) {
          const int4 v = load_cluster4(in_block(mine, q));
          sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        const float xs = p.x_scales[t0 + j];
        const int all[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < p.N) store_out(p, t0 + j, n + e, scaled(all[e], xs, p.w_scales[n + e]));
      }
    }
    __syncwarp();
    cluster_sync();                                              // nobody leaves while its sums are read
  }
  __syncthreads();
  if (s_abort) give_up_delay();                                  // let copies that may still be in flight land
  tc_fence_after();
  if (warp == 1) tmem_dealloc<1>(tmem_base, COLUMNS);
}

// ---- many tokens: pairs of blocks, 256 tokens on the MMA's M axis (128 a block), 256 outputs on its N axis (128 rows of the weight
// in each block's shared memory), tiles handed out in turn to a grid of one pair for two SMs.
constexpr int PAIR_THREADS = 320;      // producer warp, MMA warp, eight epilogue warps
constexpr int PAIR_STAGES = 6;
constexpr int HALF_BYTES = 128 * BK;   // an operand's half of a stage
constexpr size_t PAIR_SMEM = 1024 + (size_t)PAIR_STAGES * 2 * HALF_BYTES + 8 * 128 * 4 + (2 * PAIR_STAGES + 4) * 8 + 16;

__device__ __forceinline__ void store_row32(const Product& p, long long at, const float (&v)[32], int room) {
  if (p.out_f32) {
    float* o = reinterpret_cast<float*>(p.out) + at;
    if (room >= 32 && ((uintptr_t)o & 31) == 0) {
#pragma unroll
      for (int i = 0; i < 32; i += 8)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(o + i), "f"(v[i]), "f"(v[i + 1]), "f"(v[i + 2]),
                     "f"(v[i + 3]), "f"(v[i + 4]), "f"(v[i + 5]), "f"(v[i + 6]), "f"(v[i + 7]) : "memory");
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < room) o[i] = v[i];
    }
    return;
  }
  bf16* o = reinterpret_cast<bf16*>(p.out) + at;
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  if (room >= 32 && ((uintptr_t)o & 31) == 0) {
#pragma unroll
    for (int i = 0; i < 16; i += 8)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(o + 2 * i), "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]),
                   "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7]) : "memory");
  } else if (room >= 32 && ((uintptr_t)o & 3) == 0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) reinterpret_cast<uint32_t*>(o)[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < room) o[i] = __float2bfloat16_rn(v[i]);
  }
}

// The tile'th tile: `group` tiles of tokens after one another beside the same rows of the weight, then the next rows.
__device__ __forceinline__ void tile_place(const Mapped& m, int tile, int& tt, int& tn) {
  const int per = m.group * m.tiles_n, g = tile / per, r = tile - g * per;
  const int here = min(m.group, m.tiles_t - g * m.group);
  tn = r / here;
  tt = g * m.group + (r - tn * here);
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1) product_pair_kernel(const __grid_constant__ Mapped m) {
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* ring = smem_unaligned + ((1024 - (smem_u32(smem_unaligned) & 1023)) & 1023);
  float* scales = reinterpret_cast<float*>(ring + (size_t)PAIR_STAGES * 2 * HALF_BYTES);      // [8 warps][128]
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + 8 * 128);        // used in block 0, for both
  uint64_t* empty = full + PAIR_STAGES;
  uint64_t* acc_full = empty + PAIR_STAGES;      // [2]
  uint64_t* acc_empty = acc_full + 2;            // [2], used in block 0
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  __shared__ int s_abort;

  const Product& p = m.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pairs = gridDim.x >> 1, pair = blockIdx.x >> 1;
  const int tiles = m.tiles_t * m.tiles_n, kt = (p.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < PAIR_STAGES; ++s) {
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
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();

  if (warp == 0) {
    if (elect_one()) {
      int i = 0;
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs) {
        int tt, tn;
        tile_place(m, tile, tt, tn);
        const int t0 = tt * 256 + (int)rank * 128, n0 = tn * 256 + (int)rank * 128;
        for (int k = 0; k < kt; ++k, ++i) {
          const int s = i % PAIR_STAGES;
          if (i >= PAIR_STAGES && !mbar_wait(&empty[s], (uint32_t)((i / PAIR_STAGES) - 1) & 1, 1)) { ok = false; break; }
          unsigned char* dst = ring + (size_t)s * 2 * HALF_BYTES;
          const uint32_t bar = in_block(smem_u32(&full[s]), 0);
          if (rank == 0) mbar_expect_tx(&full[s], 4 * HALF_BYTES);      // zero-filled parts of a box count too
          tma_load_2d_pair(dst, &m.x_map, k * BK, t0, bar);
          tma_load_2d_pair(dst + HALF_BYTES, &m.w_map, k * BK, n0, bar);
        }
      }
      // no block leaves before the last commits have reached it
      for (int j = max(0, i - PAIR_STAGES); j < i && ok; ++j) ok = mbar_wait(&empty[j % PAIR_STAGES], (uint32_t)(j / PAIR_STAGES) & 1, 1);
      if (!ok) s_abort = 1;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc = instr_desc(256, 256);
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
          const int s = i % PAIR_STAGES;
          ok = __all_sync(0xffffffffu, mbar_wait(&full[s], (uint32_t)(i / PAIR_STAGES) & 1, 3));
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t a = smem_desc(smem_u32(ring) + s * 2 * HALF_BYTES), b = a + (HALF_BYTES >> 4);
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
    const int quarter = warp & 3, half = warp >= 6 ? 128 : 0;      // lanes that this warp may read; its columns
    float* mine = scales + (warp - 2) * 128;
    int turn = 0;
    bool ok = true;
    for (int tile = pair; tile < tiles; tile += pairs, ++turn) {
      int tt, tn;
      tile_place(m, tile, tt, tn);
      const int t = tt * 256 + (int)rank * 128 + quarter * 32 + lane, n0 = tn * 256 + half;
      const float xs = t < p.T ? p.x_scales[t] : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + j * 32 + lane;
        mine[j * 32 + lane] = n < p.N ? p.w_scales[n] : 0.f;
      }
      __syncwarp();
      ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[turn & 1], (uint32_t)(turn >> 1) & 1, 4));
      if (!ok) break;
      tc_fence_after();
      const uint32_t at = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)((turn & 1) * 256 + half);
      for (int c = 0; c < 128; c += 32) {
        int r[32];
        float v[32];
        tmem_ld32(r, at + c);
        tmem_ld_wait();
        if (c == 96) {                                             // the accumulator is read: the MMAs may have it again
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
        if (t < p.T && n0 + c < p.N) store_row32(p, (long long)t * p.out_stride + n0 + c, v, p.N - n0 - c);
      }
      __syncwarp();
    }
    if (!ok) s_abort = 1;
  }
  __syncthreads();
  if (s_abort) give_up_delay();                                  // let copies that may still be in flight land
  cluster_sync();                                                // the other block's MMAs, commits and copies reach in here
  tc_fence_after();
  if (warp == 1) tmem_dealloc<2>(tmem_base, 512);
}

// A tensor map over rows of bytes, read in boxes of 128 bytes x `rows_of_box` rows with the 128-byte swizzle.
bool make_map(CUtensorMap* map, const void* base, long long rows, long long bytes, long long stride, int rows_of_box) {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = []() -> PFN_cuTensorMapEncodeTiled_v12000 {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess) return nullptr;
    return (PFN_cuTensorMapEncodeTiled_v12000)fn;
  }();
  if (!encode) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)bytes, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
  const cuuint32_t box[2] = {BK, (cuuint32_t)rows_of_box}, steps[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NT, int STAGES>
int launch_split(const Mapped& m, cudaStream_t stream) {
  constexpr size_t smem = 1024 + (size_t)STAGES * (W_BYTES + NT * BK) + (2 * STAGES + 1) * 8 + 16;
  static_assert(smem <= 227 * 1024, "the ring must fit one block's shared memory");
  static std::atomic<uint64_t> allowed{0};
  NHV_CUDA(nhv_allow_smem((const void*)product_split_kernel<NT, STAGES>, (int)smem, allowed), "linear_int8");
  NHV_CUDA(nhv_launch_cluster(product_split_kernel<NT, STAGES>, dim3(m.tiles_n * m.group, m.tiles_t), dim3(SPLIT_THREADS), smem, stream, m.group, m),
           "linear_int8");
  return 0;
}

int split_product(Mapped& m, int parts, cudaStream_t stream) {
  const Product& p = m.p;
  m.nt = p.T >= 256 ? 256 : (p.T + 15) / 16 * 16;
  m.tiles_t = (p.T + m.nt - 1) / m.nt;
  m.tiles_n = (p.N + 127) / 128;
  m.group = parts;
  NHV_REQUIRE(make_map(&m.w_map, p.w, p.N, p.K, p.w_stride, 128) && make_map(&m.x_map, p.x, p.T, p.K, p.x_stride, m.nt),
              "linear_int8: cannot encode the tensor maps");
  if (m.nt <= 16) return launch_split<16, 5>(m, stream);
  if (m.nt <= 32) return launch_split<32, 5>(m, stream);
  if (m.nt <= 64) return launch_split<64, 4>(m, stream);
  if (m.nt <= 128) return launch_split<128, 6>(m, stream);
  return launch_split<256, 4>(m, stream);
}

int pair_product(Mapped& m, int sms, cudaStream_t stream) {
  const Product& p = m.p;
  m.nt = 256;
  m.tiles_t = (p.T + 255) / 256;
  m.tiles_n = (p.N + 255) / 256;
  m.group = m.tiles_t < 16 ? m.tiles_t : 16;
  NHV_REQUIRE(make_map(&m.w_map, p.w, p.N, p.K, p.w_stride, 128) && make_map(&m.x_map, p.x, p.T, p.K, p.x_stride, 128),
              "linear_int8: cannot encode the tensor maps");
  const long long tiles = (long long)m.tiles_t * m.tiles_n;
  NHV_REQUIRE(tiles < (1LL << 30), "linear_int8: too many tiles");
  const int pairs = (int)(tiles < sms / 2 ? tiles : sms / 2);
  static std::atomic<uint64_t> allowed{0};
  NHV_CUDA(nhv_allow_smem((const void*)product_pair_kernel, (int)PAIR_SMEM, allowed), "linear_int8");
  NHV_CUDA(nhv_launch(product_pair_kernel, dim3(2 * pairs), dim3(PAIR_THREADS), PAIR_SMEM, stream, m), "linear_int8");
  return 0;
}

}  // namespace

// Reads and clears the error word (0: no bounded wait ever ran out).  Synchronises the device.
NHV_API int nhv_gemm_int8_error() { return nhv_wait_error_take(); }
// The device address of the error word, for kernels that report it with the step's result.
NHV_API void* nhv_gemm_int8_error_word() { return nhv_wait_error_address(); }

NHV_API int nhv_gemm_int8(void* out, int out_dtype, long long out_stride, const void* x, long long x_stride, const float* x_scales,
                          const void* w, long long w_stride, const float* w_scales, int T, int N, int K, int sms, int way, cudaStream_t stream) {
  if (T == 0 || N == 0) return 0;
  NHV_REQUIRE(T > 0 && N > 0 && K > 0 && K <= 131071, "linear_int8: a sum over 1 to 131,071 products is exact in 32 bits, not over %d", K);
  NHV_REQUIRE(out && x && w && x_scales && w_scales && (out_dtype == NHV_F32 || out_dtype == NHV_BF16), "linear_int8: bad arguments");
  const Product p = {(const int8_t*)x, (const int8_t*)w, x_scales, w_scales, out, x_stride, w_stride, out_stride, T, N, K, out_dtype == NHV_F32};
  const bool aligned = ((uintptr_t)x | (uintptr_t)w | (uintptr_t)x_stride | (uintptr_t)w_stride) % 16 == 0;
  if (aligned && way != 1) {
    Mapped m;
    m.p = p;
    if (way == 3 || (way == 0 && T > 256)) return pair_product(m, sms, stream);
    const int tiles = (N + 127) / 128 * ((T + 255) / 256), kt = (K + BK - 1) / BK;
    int parts = way >= 10 ? way - 10 : 2 * sms / tiles;
    parts = parts < 1 ? 1 : parts > 8 ? 8 : parts;
    return split_product(m, parts < kt ? parts : kt, stream);
  }
  const int rows = (T + TILE - 1) / TILE;
  NHV_REQUIRE(rows <= 65535, "linear_int8: %d tokens are more than a call takes", T);
  NHV_CUDA(nhv_launch(product_any_kernel, dim3((N + TILE - 1) / TILE, rows), dim3(256), 0, stream, p), "linear_int8");
  return 0;
}
