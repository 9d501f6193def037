// Attention with scored keys for requests that bring many rows (a row: a new token and a query head of one KV head), bfloat16, on
// the 5th-generation tensor cores: tcgen05.mma with the accumulators in tensor memory, operands brought by TMA.
//
// The rows' pass: O = softmax(Q K^T) V, and each row's log-sum.  A block owns two tiles of up to 128 rows (whole tokens; heads above
// 128: one tile) of a KV head and walks the keys in tiles of 64.  Warp 0, one lane: TMA, keys and values through one ring of
// stages, straight from the pages, in boxes of as many rows as divide the page size and 64.  Warp 1, one lane: the MMAs,
// S = Q K^T into one of two buffers a tile of rows, and O += P V.  Warps 4-7 and 8-11: one thread per row of the first and the second
// tile; it reads its row of S, takes maximum and exponentials, writes P (bfloat16) over S.  The next S is made while this one is in
// the softmax.  O is rescaled only when a row's maximum grew by more than 2^8; then, and only then, the product before is waited for.
//   P is rounded to the type that the MMA takes beside V.  With the output's own rounding that is an error of 2.1e-3 to 2.3e-3 of the
//   output against 64 bits, where an output rounded once has 1.6e-3 to 1.7e-3; the remainder as a second part would be half as many MMAs
//   again and two instructions more for a pair, where the pass waits for instructions as it is.
//   Tried: tiles of 128 keys with one buffer of S (the softmax then waits for P V and the next Q K^T, 1,024 cycles of a step of 4,430:
//   385 us for 1,024 tokens behind 16,384 keys); the same with two threads a row (458 us: the threads of a row meet for the maximum).
//   Where the grid would leave SMs idle the keys are split over blocks, whose sums a small kernel joins.
// The keys' pass: w[j] = sum over the rows that see j of exp2(s - log-sum).  S^T = K Q^T with the keys as M: a lane of tensor
// memory is a key and its columns are rows, so a thread adds up its key's weights with no exchange at all.  The block's keys stay
// in shared memory, the tiles of rows stream through a ring.  Under the causal mask a request's first keys are seen by all rows
// and its last by few; so the rows are cut into chunks, a block per (key tile, chunk), and the chunks' sums added in their order.
// Making S a second time costs 2 D operations a pair where keeping P would write and read 4 bytes a pair, eight times the time.
//
// What bounds them: an exponential a pair in each pass (16 a cycle and SM, where the MMAs make 32 pairs a cycle in the rows' pass with
// heads of 128 and 64 in the keys'), and beside it the turns between MMAs and softmax.  1,024 tokens behind 16,384 keys, 32 heads on 8
// of 128, 553 million pairs: 137 us of exponentials in each; rows 292 us (970 TFLOP/s of 4 D a pair), keys 206 us (690 of 2 D).  A prompt
// of 2,048 tokens, whose 264 blocks fill the SMs badly: 53 and 39 us.
//
// A key out of sight may hold anything.  Its score is replaced.  Its value would reach the rows that do not see it as 0 times no
// number, so tiles of which some row sees a part have their values looked through: what is not finite is taken out of shared
// memory, and the rows that do see it get it back at the end, from the pages.
//
// Every wait on an mbarrier is bounded: one that runs out sets the file's error word, the roles leave their loops, the producer
// waits (bounded) for its copies in flight, and the block frees its tensor memory and returns.
#define NHV_WAIT_LIMIT (1u << 22)
#include "nhv_async.cuh"
#include "nhv_scored.cuh"

namespace {

typedef __nv_bfloat16 bf16;
constexpr int BM = 128;                          // rows of a tile = lanes of tensor memory
constexpr float RESCALE_STEP = 8.0f;             // log2 units
constexpr int SMS = 148;

template <int DB> struct Rows {                  // DB: blocks of 64 elements (128 bytes) of a head
  static constexpr int NQ = DB <= 2 ? 2 : 1;     // tiles of rows a block
  static constexpr int BN = 64;                  // keys of a tile
  static constexpr int THREADS = 128 + NQ * 128;
  static constexpr int Q_BYTES = DB * BM * 128, STAGE = DB * BN * 128;
  static constexpr int STAGES = DB == 1 ? 12 : DB == 2 ? 10 : 5;
  static constexpr int SMEM = 1024 + 1024 + NQ * Q_BYTES + STAGES * STAGE;       // barriers and notes, alignment, tiles
  static constexpr uint32_t S_COL = 0, O_COL = NQ * 2 * BN;      // two buffers of S a tile of rows
  static constexpr uint32_t TMEM_COLS = 512;
};
template <int DB> struct Keys {
  static constexpr int BN = 128;                 // rows of a tile = columns of S^T
  static constexpr int THREADS = 64 + 256;
  static constexpr int K_BYTES = DB * BM * 128, STAGE = DB * BN * 128;
  static constexpr int STAGES = DB == 1 ? 4 : DB == 2 ? 2 : 1;     // two blocks an SM (tensor memory has room for two), above 128 one
  static constexpr int SMEM = 1024 + 1024 + 1024 + K_BYTES + STAGES * STAGE;
  static constexpr uint32_t TMEM_COLS = 256;     // two buffers
};

struct alignas(64) LongArgs {
  CUtensorMap kv_map;       // the pool as [n_pages * 2 * nkv * page_size, d], boxes of 64 columns x `box` rows
  CUtensorMap q_map;        // q as [n_tokens, nq, d], boxes of 64 columns x G heads x tokens of a tile
  ScoredArgs a;
  NhvScoreCap cap;
  float scale_log2;
  ScoredParts parts;
  int key_tiles;
  int tokens, box;          // tokens of a tile of rows; rows of a TMA box of the pages
};

// ---- tensor memory and tcgen05
__device__ __forceinline__ void tmem_alloc(uint32_t* slot_in_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(slot_in_smem)), "r"(ncols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
// One lane of a converged warp.  MMAs are issued under this and not under `lane == 0`, with what they are made from the same in every
// lane by a shuffle: their operands live in the warp's uniform registers, and where the compiler cannot see that a value is the
// same in all lanes, each MMA took about 137 cycles to issue, whatever its size (506 -> 335 us for the rows of 1,024 tokens behind
// 16,384 keys).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void tc_mma(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
// The same with the A operand in tensor memory (one row per lane, two bfloat16 per 32-bit column).
__device__ __forceinline__ void tc_mma_a_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
// 32 consecutive columns of this thread's lane (no wait: tmem_ld_wait() before the values are used)
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t (&r)[32], uint32_t taddr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t (&r)[16], uint32_t taddr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// Shared-memory matrix descriptor, 128-byte swizzle.  K-major operand (Q, K): rows of 128 bytes, groups of 8 rows 1024 bytes apart
// (stride offset), the leading offset unused.  MN-major operand (V as it lies in the cache: a row of 128 bytes holds 64 elements of
// one key): the stride offset is the step between groups of 8 keys, the leading offset the step between blocks of 64 elements.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t leading_bytes, uint32_t stride_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFF) >> 4);
  d |= (uint64_t)((leading_bytes >> 4) & 0x3FFF) << 16;
  d |= (uint64_t)((stride_bytes >> 4) & 0x3FFF) << 32;
  d |= (uint64_t)1 << 46;                            // descriptor version of this architecture
  d |= (uint64_t)2 << 61;                            // 128-byte swizzle
  return d;
}
// Instruction descriptor: bf16 x bf16 -> fp32, A K-major, M x N; B K-major or MN-major.
__device__ __forceinline__ uint32_t instr_desc(int m, int n, bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn_major ? (1u << 16) : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ f32x2 f2_add(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// 256 threads meet.
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 256;\n" ::"r"(id) : "memory"); }
// 32 scores capped (see nhv_cap_tile): where a warp's are all small, two at a time by the polynomial.  A lane that does not count has no
// say in that, or the last bits of the others would go by what lies about in shared memory and in pages' unused slots.
__device__ __forceinline__ void cap32(uint32_t (&sr)[32], const NhvScoreCap& c, bool counts) {
  float m0 = 0.f, m1 = 0.f;
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    m0 = max3(m0, fabsf(__uint_as_float(sr[i])), fabsf(__uint_as_float(sr[i + 1])));
    m1 = max3(m1, fabsf(__uint_as_float(sr[i + 2])), fabsf(__uint_as_float(sr[i + 3])));
  }
  if (__all_sync(0xffffffffu, !counts || fmaxf(m0, m1) <= c.small)) {
    const f32x2 z2 = f2_pack(c.z, c.z), k0 = f2_pack(c.c[0], c.c[0]), k1 = f2_pack(c.c[1], c.c[1]), k2 = f2_pack(c.c[2], c.c[2]),
                k3 = f2_pack(c.c[3], c.c[3]), k4 = f2_pack(c.c[4], c.c[4]);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const f32x2 z = f2_mul(f2_pack(__uint_as_float(sr[i]), __uint_as_float(sr[i + 1])), z2), t = f2_mul(z, z);
      float x, y;
      f2_unpack(f2_mul(z, f2_fma(f2_fma(f2_fma(f2_fma(k4, t, k3), t, k2), t, k1), t, k0)), x, y);
      sr[i] = __float_as_uint(x);
      sr[i + 1] = __float_as_uint(y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float x = __uint_as_float(sr[i]), y = __uint_as_float(sr[i + 1]);
      nhv_cap_scores<true>(x, y, c);
      sr[i] = __float_as_uint(x);
      sr[i + 1] = __float_as_uint(y);
    }
  }
}

// What few tiles need, out of the way of what all need: scores capped and masked where they lie in tensor memory (32 columns at a
// time); a key at or above `end` of the row's own, or without a page, gets -inf.
template <int BN>
__device__ __noinline__ void change_scores(uint32_t s_addr, const NhvScoreCap& cap, bool masked, bool missing, int key0, int row_hi, int total, const int* table,
                                           int page_size, int n_pages) {
#pragma unroll 1
  for (int c = 0; c < BN; c += 32) {
    uint32_t sr[32];
    tmem_ld32_nowait(sr, s_addr + c);
    tmem_ld_wait();
    uint32_t gone = 0;
    if (masked) {
      if (missing)
        for (int i = 0; i < 32; ++i) {
          const int page = table[min(key0 + c + i, total - 1) / page_size];
          if (page < 0 || page >= n_pages) gone |= 1u << i;
        }
#pragma unroll
      for (int i = 0; i < 32; ++i) gone |= key0 + c + i > row_hi ? 1u << i : 0u;
    }
    if (cap.in != 0.f) {
#pragma unroll
      for (int i = 0; i < 32; ++i) sr[i] = gone >> i & 1u ? 0u : sr[i];
      cap32(sr, cap, true);
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) sr[i] = gone >> i & 1u ? 0xFF800000u : sr[i];
    tmem_st32(s_addr + c, sr);
  }
  tmem_st_wait();
}
// A thread group's pass over a tile of values in shared memory: rows that are no key of the request become zeros, and, with
// `finite`, so does what is not finite, each such key noted in bad_keys[2].
template <int DB, int BN>
__device__ __noinline__ void clean_values(unsigned char* v, uint32_t* bad_keys, bool finite, bool missing, int key0, int total, const int* table,
                                          int page_size, int n_pages) {
  for (int id = threadIdx.x & 127; id < BN * DB * 8; id += 128) {
    const int row = id / (DB * 8), rem = id - row * (DB * 8), at_key = min(key0 + row, total - 1);
    uint4* at = reinterpret_cast<uint4*>(v + (rem >> 3) * (BN * 128) + row * 128 + ((rem & 7) << 4));
    const int page = missing ? table[at_key / page_size] : 0;
    if (key0 + row >= total || page < 0 || page >= n_pages) {
      *at = make_uint4(0, 0, 0, 0);
    } else if (finite) {
      uint4 x = *at;
      bool bad = false;
      x.x = finite_pair(x.x, bad); x.y = finite_pair(x.y, bad); x.z = finite_pair(x.z, bad); x.w = finite_pair(x.w, bad);
      if (bad) {
        atomicOr(&bad_keys[row >> 5], 1u << (row & 31));
        *at = x;
      }
    }
  }
  fence_async_smem();
}
// Values taken out above, back to a row that sees them: p v, of what is not finite in v, added to O in tensor memory.  `notes`: the 8 x 2
// words of keys, from key `key0` on in tiles of BN.
template <int DB, int BN>
__device__ __noinline__ void return_values(uint32_t o_addr, const ScoredArgs& a, const uint32_t* notes, int seq, int kvh, int head, int token, int key0,
                                           int row_hi, float m, float scale_log2) {
#pragma unroll 1
  for (int c0 = 0; c0 < DB * 64; c0 += 32) {
    uint32_t o[32];
    tmem_ld32_nowait(o, o_addr + c0);
    tmem_ld_wait();
    for (int w = 0; w < 16; ++w)
      for (uint32_t bits = notes[w]; bits; bits &= bits - 1) {
        const int key = key0 + (w >> 1) * BN + (w & 1) * 32 + __ffs(bits) - 1;
        if (key > row_hi) continue;
        const long long k_at = key_row(a, seq, key, kvh, 0), v_at = key_row(a, seq, key, kvh, 1);
        if (k_at < 0) continue;
        const bf16* qr = (const bf16*)a.q + (size_t)token * a.q_stride + (size_t)head * a.d;
        float s = 0.f;
        for (int e = 0; e < a.d; ++e) s = fmaf(to_f32(qr[e]), to_f32(((const bf16*)a.pages)[k_at + e]), s);
        if (a.softcap > 0.f) s = a.softcap * tanhf(s * a.scale / a.softcap) * SA_LOG2E;
        else s *= scale_log2;
        const float weight = scored_exp2(s + (m == -INFINITY ? 0.f : -m));
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float x = c0 + i < a.d ? to_f32(((const bf16*)a.pages)[v_at + c0 + i]) : 0.f;
          if (!(fabsf(x) < INFINITY)) o[i] = __float_as_uint(fmaf(weight, x, __uint_as_float(o[i])));
        }
      }
    __syncwarp();
    tmem_st32(o_addr + c0, o);
  }
  tmem_st_wait();
}

// Where tiles of BN keys lie: a lane per box of rows, which lie in one page each.  A lane asks for the page of its box a tile ahead (one
// lane that looked each tile up and then sent for it took 1,900 cycles a tile).  Boxes at or behind `total` and those without a page
// bring some other row: their scores are replaced and their values cleared.
template <int BN>
struct BoxWalk {
  const int* table;
  int at, off, last_at, last_off, key, total, page;        // page index and place of the lane's box, and of the request's last box
  int page_size, step;
  __device__ __forceinline__ BoxWalk(const LongArgs& p, int seq, int key0, int total_, int lane)
      : table(p.a.block_table + (size_t)seq * p.a.bt_stride), total(total_), page_size(p.a.page_size), step(p.box < BN ? p.box : BN) {
    key = key0 + lane * step;
    at = key / page_size;
    off = key - at * page_size;
    last_at = (total - 1) / page_size;
    last_off = (total - 1 - last_at * page_size) / step * step;
    ask();
  }
  __device__ __forceinline__ void ask() { page = table[key < total ? at : last_at]; }
  // the pool's row of the box asked for
  __device__ __forceinline__ int row(const LongArgs& p, int kvh) const {
    const int use = page < 0 || page >= p.a.n_pages ? 0 : page;
    return (use * 2 * p.a.nkv + kvh) * page_size + (key < total ? off : last_off);
  }
  __device__ __forceinline__ void next() {                  // asks for the box of the next tile
    key += BN;
    off += BN;
    while (off >= page_size) {
      off -= page_size;
      ++at;
    }
    ask();
  }
};
// The warp's copy of a tile of keys (plane 0) or values (plane 1) into one stage.
template <int DB, int BN>
__device__ __forceinline__ void load_tile(unsigned char* stage, const LongArgs& p, int row, int plane, uint64_t* bar, int lane) {
  const int step = p.box < BN ? p.box : BN;
  if (step == BN) {                                         // one box, one lane, with what it needs the same in all
    const int y = __shfl_sync(0xffffffffu, row, 0) + plane * p.a.nkv * p.a.page_size;
    if (elect_one()) {
      mbar_expect_tx(bar, DB * BN * 128);
#pragma unroll
      for (int b = 0; b < DB; ++b) tma_load_2d(stage + b * (BN * 128), &p.kv_map, b * 64, y, bar);
    }
  } else {
    if (lane == 0) mbar_expect_tx(bar, DB * BN * 128);
    __syncwarp();
    if (lane * step < BN) {
#pragma unroll
      for (int b = 0; b < DB; ++b) tma_load_2d(stage + b * (BN * 128) + lane * step * 128, &p.kv_map, b * 64, row + plane * p.a.nkv * p.a.page_size, bar);
    }
  }
  __syncwarp();
}
template <int DB>
__device__ __forceinline__ void load_rows(unsigned char* stage, const LongArgs& p, int token, int kvh, int G, uint64_t* bar) {
  mbar_expect_tx(bar, DB * p.tokens * G * 128);
#pragma unroll
  for (int b = 0; b < DB; ++b) tma_load_3d(stage + b * (BM * 128), &p.q_map, b * 64, kvh * G, token, bar);
}

template <int DB, bool CAP>
__global__ void __launch_bounds__(Rows<DB>::THREADS, 1) scored_rows_tcgen05_kernel(const __grid_constant__ LongArgs p) {
  using C = Rows<DB>;
  constexpr int NQ = C::NQ, BN = C::BN, STAGES = C::STAGES;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_raw);
  uint64_t* full = bars;                   // [STAGES]
  uint64_t* empty = bars + 12;             // [STAGES]
  uint64_t* s_full = bars + 24;            // [NQ][2]
  uint64_t* p_ready = bars + 28;           // [NQ][2]: by buffer, since the rows may be a tile ahead of the products
  uint64_t* o_full = bars + 32;            // [NQ]: after every product
  uint64_t* o_last = bars + 34;            // [NQ]: after the last one
  uint64_t* q_full = bars + 36;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 37);
  int* s_abort = reinterpret_cast<int*>(bars + 38);
  int* s_missing = reinterpret_cast<int*>(bars + 39);
  uint32_t* s_bad = reinterpret_cast<uint32_t*>(bars + 40);       // [8 tiles][2]: keys whose values are not all finite
  const uint32_t raw = smem_u32(smem_raw);
  unsigned char* tiles = smem_raw + (((raw + 1024 + 1023u) & ~1023u) - raw);
  unsigned char* q_s = tiles;                          // [NQ][Q_BYTES]
  unsigned char* kv_s = q_s + NQ * C::Q_BYTES;         // [STAGES][STAGE]

  const ScoredArgs& a = p.a;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int q = 0; q < NQ; ++q) {
      mbar_init(&s_full[2 * q], 1);
      mbar_init(&s_full[2 * q + 1], 1);
      mbar_init(&p_ready[2 * q], 128);
      mbar_init(&p_ready[2 * q + 1], 128);
      mbar_init(&o_full[q], 1);
      mbar_init(&o_last[q], 1);
    }
    mbar_init(q_full, 1);
    *s_abort = 0;
    *s_missing = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"((uint64_t)&p.kv_map) : "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"((uint64_t)&p.q_map) : "memory");
  }
  if (threadIdx.x < 16) s_bad[threadIdx.x] = 0;
  if (warp == 1) tmem_alloc(tmem_slot, C::TMEM_COLS);
  pdl_prologue();

  // which request, which rows, which keys: within a request the last tokens, which see the most, come first
  const int G = a.nq / a.nkv, kvh = blockIdx.x, per_block = NQ * p.tokens;
  int tile = blockIdx.y;
  const int seq = find_tile(a, per_block, tile);
  int first = 0, n = 0, total = 0, t0 = 0, key_begin = 0;
  int nt[2] = {0, 0};                                  // tiles of keys that the rows of tile q see, of this block's part
  if (seq >= 0) {
    first = a.cu_q[seq];
    n = a.cu_q[seq + 1] - first;
    total = min(a.kv_len[seq], a.max_keys);
    t0 = ((n + per_block - 1) / per_block - 1 - tile) * per_block;
    key_begin = (int)blockIdx.z * p.parts.split_tiles * BN;
    for (int q = 0; q < NQ; ++q) {
      const int t_last = min(t0 + (q + 1) * p.tokens, n) - 1;
      if (t_last < t0 + q * p.tokens) continue;
      const int seen = total - n + t_last + 1 - key_begin;
      nt[q] = seen <= 0 ? 0 : min((seen + BN - 1) / BN, p.parts.split_tiles);
    }
    const int* table = a.block_table + (size_t)seq * a.bt_stride;
    const int page_end = (min(key_begin + max(nt[0], nt[1]) * BN, total) + a.page_size - 1) / a.page_size;
    for (int i = key_begin / a.page_size + threadIdx.x; i < page_end; i += C::THREADS)
      if (table[i] < 0 || table[i] >= a.n_pages) *s_missing = 1;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const int n_tiles = __shfl_sync(0xffffffffu, max(nt[0], nt[1]), 0);
  nt[0] = __shfl_sync(0xffffffffu, nt[0], 0);
  nt[1] = __shfl_sync(0xffffffffu, nt[1], 0);

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (n_tiles > 0) {
      BoxWalk<BN> walk(p, seq, key_begin, total, lane);
      if (lane == 0) {
        mbar_expect_tx(q_full, (uint32_t)((nt[0] > 0) + (nt[1] > 0)) * DB * p.tokens * G * 128);
        for (int q = 0; q < NQ; ++q)
          if (nt[q] > 0) {
#pragma unroll
            for (int b = 0; b < DB; ++b) tma_load_3d(q_s + q * C::Q_BYTES + b * (BM * 128), &p.q_map, b * 64, kvh * G, first + t0 + q * p.tokens, q_full);
          }
      }
      __syncwarp();
      bool ok = true;
      int sent = 0;
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int row = walk.row(p, kvh);
        walk.next();
        for (int plane = 0; plane < 2 && ok; ++plane) {
          const int i = 2 * j + plane, st = i % STAGES;
          if (i >= STAGES) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], (uint32_t)(i / STAGES - 1) & 1, 1));
          if (!ok) break;
          load_tile<DB, BN>(kv_s + st * C::STAGE, p, row, plane, &full[st], lane);
          sent = i + 1;
        }
      }
      if (!ok && lane == 0) {
        *s_abort = 1;
        mbar_wait(q_full, 0, 2);
        for (int i = max(0, sent - STAGES); i < sent; ++i) mbar_wait(&full[i % STAGES], (uint32_t)(i / STAGES) & 1, 2);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (n_tiles > 0) {
      const uint32_t idesc_s = instr_desc(BM, BN, false), idesc_o = instr_desc(BM, DB * 64, true);
      const uint64_t q_desc = smem_desc(smem_u32(q_s), 16, 1024);
      const uint64_t k_desc = smem_desc(smem_u32(kv_s), 16, 1024);
      const uint64_t v_desc = smem_desc(smem_u32(kv_s), BN * 128, 1024);
      // every lane waits, and all go on or none
      auto reached = [&](uint64_t* bar, uint32_t parity, int code) -> bool { return __all_sync(0xffffffffu, mbar_wait(bar, parity, code)); };
      bool ok = reached(q_full, 0, 3);
      tc_fence_after();
      auto stage_ready = [&](int i) { return reached(&full[i % STAGES], (uint32_t)(i / STAGES) & 1, 4); };
      auto first_product = [&](int q, int j) {
        if (!elect_one()) return;
        const uint64_t kd = k_desc + (uint64_t)(((2 * j) % STAGES) * (C::STAGE >> 4)), qd = q_desc + (uint64_t)(q * (C::Q_BYTES >> 4));
#pragma unroll
        for (int kk = 0; kk < DB * 4; ++kk)
          tc_mma(tmem_base + C::S_COL + (2 * q + (j & 1)) * BN, qd + (uint64_t)(((kk >> 2) * (BM * 128) + (kk & 3) * 32) >> 4),
                 kd + (uint64_t)(((kk >> 2) * (BN * 128) + (kk & 3) * 32) >> 4), idesc_s, kk > 0 ? 1u : 0u);
        tc_commit(&s_full[2 * q + (j & 1)]);
      };
      auto second_product = [&](int q, int j) {
        if (!elect_one()) return;
        const uint64_t vd = v_desc + (uint64_t)(((2 * j + 1) % STAGES) * (C::STAGE >> 4));
        const uint32_t pa = tmem_base + C::S_COL + (2 * q + (j & 1)) * BN;       // P lies over the first half of S
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk)                          // 8 columns of P and 16 rows of V per 16 keys
          tc_mma_a_tmem(tmem_base + C::O_COL + q * (DB * 64), pa + kk * 8, vd + (uint64_t)((kk * 16 * 128) >> 4), idesc_o,
                        (j > 0 || kk > 0) ? 1u : 0u);
        tc_commit(&o_full[q]);
        if (j == nt[q] - 1) tc_commit(&o_last[q]);
      };
      if (ok) ok = stage_ready(0);
      if (ok) {
        tc_fence_after();
        for (int q = 0; q < NQ; ++q)
          if (nt[q] > 0) first_product(q, 0);
        if (elect_one()) tc_commit(&empty[0]);
        __syncwarp();
      }
      for (int j = 0; j < n_tiles && ok; ++j) {
        // the next tile's S goes to the other buffer, whose P the products before have read
        if (j + 1 < n_tiles) {
          ok = stage_ready(2 * j + 2);
          if (!ok) break;
          tc_fence_after();
          for (int q = 0; q < NQ; ++q)
            if (j + 1 < nt[q]) first_product(q, j + 1);
          if (elect_one()) tc_commit(&empty[(2 * j + 2) % STAGES]);
          __syncwarp();
        }
        ok = stage_ready(2 * j + 1);
        for (int q = 0; q < NQ && ok; ++q) {
          if (j >= nt[q]) continue;
          ok = reached(&p_ready[2 * q + (j & 1)], (uint32_t)(j >> 1) & 1, 5);
          if (!ok) break;
          tc_fence_after();
          second_product(q, j);
        }
        if (ok && elect_one()) tc_commit(&empty[(2 * j + 1) % STAGES]);
        __syncwarp();
      }
      if (!ok) *s_abort = 1;
    }
    __syncwarp();
  } else if (warp >= 4 && seq >= 0) {
    // ------------------------------------------------------------------ softmax and output: a thread per row
    const int q = (warp - 4) >> 2, quarter = warp & 3, R = quarter * 32 + lane;
    const int tq = R / G, g = R - tq * G, token = t0 + q * p.tokens + tq;
    const bool valid = tq < p.tokens && token < n;
    const int row_hi = valid ? total - n + token : -1;                 // the newest key that the row sees
    const int all_hi = total - n + t0 + q * p.tokens;                  // every row of the tile sees keys up to here
    const int tiles_q = nt[q];
    const bool missing = *s_missing != 0;
    const int* table = a.block_table + (size_t)seq * a.bt_stride;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_base = lane_addr + C::S_COL + q * 2 * BN, o_addr = lane_addr + C::O_COL + q * (DB * 64);
    float m = -INFINITY, l = 0.f;
    // the first tile of which some row of the block does not see all; the notes on values begin there
    const int first_edge = max(0, total - n + t0 + 1 - key_begin) / BN;
    bool ok = true;
    const f32x2 scale2 = f2_pack(p.scale_log2, p.scale_log2);
    for (int j = 0; j < tiles_q; ++j) {
      const int key0 = key_begin + j * BN;
      const uint32_t s_addr = s_base + (j & 1) * BN;
      // Values that some row of the block does not see: the first tile's group looks them through for both, whose product comes first.
      if ((missing || key0 + BN - 1 > total - n + t0) && (q == 0 || j >= nt[0])) {
        const int st = (2 * j + 1) % STAGES;
        ok = __all_sync(0xffffffffu, mbar_wait(&full[st], (uint32_t)((2 * j + 1) / STAGES) & 1, 7));
        if (!ok) break;
        clean_values<DB, BN>(kv_s + st * C::STAGE, &s_bad[((j - first_edge) & 7) * 2], j >= first_edge, missing, key0, total, table, a.page_size, a.n_pages);
      }
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[2 * q + (j & 1)], (uint32_t)(j >> 1) & 1, 6));
      if (!ok) break;
      tc_fence_after();
      const bool masked = key0 + BN - 1 > all_hi || missing;           // some row does not see some key of the tile
      if (masked) change_scores<BN>(s_addr, p.cap, masked, missing, key0, row_hi, total, table, a.page_size, a.n_pages);
      uint32_t sr[BN / 32][32];
#pragma unroll
      for (int c = 0; c < BN / 32; ++c) tmem_ld32_nowait(sr[c], s_addr + c * 32);
      tmem_ld_wait();
      if (CAP && !masked) {
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) cap32(sr[c], p.cap, valid);
      }
      float mx0 = max3(__uint_as_float(sr[0][0]), __uint_as_float(sr[0][1]), __uint_as_float(sr[0][2]));
      float mx1 = max3(__uint_as_float(sr[0][3]), __uint_as_float(sr[0][4]), __uint_as_float(sr[0][5]));
#pragma unroll
      for (int i = 6; i + 3 < BN; i += 4) {
        mx0 = max3(mx0, __uint_as_float(sr[i >> 5][i & 31]), __uint_as_float(sr[(i + 1) >> 5][(i + 1) & 31]));
        mx1 = max3(mx1, __uint_as_float(sr[(i + 2) >> 5][(i + 2) & 31]), __uint_as_float(sr[(i + 3) >> 5][(i + 3) & 31]));
      }
      const float mx = max3(mx0, mx1, fmaxf(__uint_as_float(sr[BN / 32 - 1][30]), __uint_as_float(sr[BN / 32 - 1][31]))) * p.scale_log2;
      const bool grow = mx > m + RESCALE_STEP;                         // also the first keys a row sees
      if (__any_sync(0xffffffffu, grow)) {
        float alpha = 1.f;
        if (grow) {
          alpha = scored_exp2(m - mx);                                 // 0 when the row had seen nothing
          m = mx;
          l *= alpha;
        }
        if (j > 0) {
          // the product before must be complete (the one before that is, or this S would not be: a parity tells the two apart)
          ok = __all_sync(0xffffffffu, mbar_wait(&o_full[q], (uint32_t)(j - 1) & 1, 8));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c0 = 0; c0 < DB * 64; c0 += 16) {
            uint32_t o[16];
            tmem_ld16(o, o_addr + c0);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st16(o_addr + c0, o);
          }
        }
      }
      const float neg_ref = m == -INFINITY ? 0.f : -m;
      const f32x2 ref2 = f2_pack(neg_ref, neg_ref);
      f32x2 l2[4] = {0ull, 0ull, 0ull, 0ull};
      uint32_t pk[BN / 2];
#pragma unroll
      for (int i = 0; i < BN; i += 2) {
        float x, y;
        f2_unpack(f2_fma(f2_pack(__uint_as_float(sr[i >> 5][i & 31]), __uint_as_float(sr[i >> 5][(i & 31) + 1])), scale2, ref2), x, y);
        x = scored_exp2(x);
        y = scored_exp2(y);
        pk[i >> 1] = pack_bf16(x, y);
        l2[(i >> 1) & 3] = f2_add(l2[(i >> 1) & 3], f2_pack(x, y));     // the row's sum in fp32, before the rounding to bfloat16
      }
      tmem_st32(s_addr, pk);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_ready[2 * q + (j & 1)]);
      l += f2_sum(f2_add(l2[0], l2[1]), f2_add(l2[2], l2[3]));
    }
    if (ok && tiles_q > 0) ok = __all_sync(0xffffffffu, mbar_wait(&o_last[q], 0, 8));
    if (ok) {
      tc_fence_after();
      // The notes on values: made before the products that o_full covers.  The other group may be noting keys that no row of this tile
      // sees, so lanes may read different words; what follows is the whole warp's business and takes one decision.
      bool any_bad = false;
      for (int i = 0; i < 16; ++i) any_bad |= *(volatile uint32_t*)&s_bad[i] != 0;
      if (__any_sync(0xffffffffu, any_bad) && tiles_q > 0)
        return_values<DB, BN>(o_addr, a, s_bad, seq, kvh, kvh * G + g, first + token, key_begin + first_edge * BN, row_hi, m, p.scale_log2);
      const size_t row = (size_t)kvh * a.n_tokens * G + (size_t)(first + token) * G + g;
      const bool whole = p.parts.splits == 1;
      float inv = 1.f;
      if (whole) {
        const float sink = a.sinks && valid ? a.sinks[kvh * G + g] * SA_LOG2E : -INFINITY;
        float ref = fmaxf(m, sink);
        if (ref == -INFINITY) ref = 0.f;
        // the sink: one more term of the sum
        const float f = scored_exp2(m - ref), sum = fmaf(l, f, scored_exp2(sink - ref));
        inv = sum == 0.f ? 0.f : f / sum;
        if (valid) a.lse[row] = sum == 0.f ? INFINITY : ref + log2f(sum);
      } else if (valid) {
        float* ml = p.parts.ml + ((size_t)blockIdx.z * a.nkv * a.n_tokens * G + row) * 2;
        ml[0] = m;
        ml[1] = l;
      }
      bf16* dst = (bf16*)a.out + (size_t)(first + token) * a.out_stride + (size_t)(kvh * G + g) * a.d;
      float* part = p.parts.o + ((size_t)blockIdx.z * a.nkv * a.n_tokens * G + row) * a.d;
#pragma unroll 1
      for (int c0 = 0; c0 < DB * 64; c0 += 32) {
        uint32_t o[32];
        if (tiles_q > 0) {
          tmem_ld32_nowait(o, o_addr + c0);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (valid && whole) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 x;
            x.x = pack_bf16(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
            x.y = pack_bf16(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
            x.z = pack_bf16(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv);
            x.w = pack_bf16(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv);
            if (c0 + i < a.d) *reinterpret_cast<uint4*>(dst + c0 + i) = x;
          }
        } else if (valid) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            if (c0 + i < a.d)
              *reinterpret_cast<uint4*>(part + c0 + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
        __syncwarp();
      }
    } else {
      *s_abort = 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

template <int DB, bool CAP>
__global__ void __launch_bounds__(Keys<DB>::THREADS, DB <= 2 ? 2 : 1) scored_keys_tcgen05_kernel(const __grid_constant__ LongArgs p) {
  using C = Keys<DB>;
  constexpr int STAGES = C::STAGES;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_raw);
  uint64_t* full = bars;                   // [STAGES]
  uint64_t* empty = bars + 4;              // [STAGES]
  uint64_t* s_full = bars + 8;             // [2]
  uint64_t* s_free = bars + 10;            // [2]
  uint64_t* k_full = bars + 12;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 14);
  int* s_abort = reinterpret_cast<int*>(bars + 15);
  float* s_part = reinterpret_cast<float*>(bars + 32);             // [128]
  float* s_lse = reinterpret_cast<float*>(smem_raw + 1024);        // [2][128], negated
  const uint32_t raw = smem_u32(smem_raw);
  unsigned char* tiles = smem_raw + (((raw + 2048 + 1023u) & ~1023u) - raw);
  unsigned char* k_s = tiles;
  unsigned char* q_s = k_s + C::K_BYTES;               // [STAGES][STAGE]

  const ScoredArgs& a = p.a;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // Blocks without work (requests of unlike length, chunks that see nothing of a tile) leave before they take tensor memory.  The others
  // have taken theirs when they let the next kernel in, so that none of this kernel's blocks can wait for what that one holds.
  pdl_wait();
  const int G = a.nq / a.nkv, kvh = blockIdx.x, seq = blockIdx.z;
  const int chunk = blockIdx.y / p.key_tiles, key0 = (blockIdx.y - chunk * p.key_tiles) * BM;
  const int first = a.cu_q[seq], n = a.cu_q[seq + 1] - first, total = min(a.kv_len[seq], a.max_keys);
  if (key0 >= total || !scored_takes(a, n)) return;
  int begin = 0, end = 0;
  chunk_range(p.parts, n, G, total, key0, chunk, begin, end);
  if (begin >= end && p.parts.chunks > 1) return;
  // Rows of a stage behind a tile's last (groups that do not divide 128) are never copied to: zeros, whose weights the log-sum of +inf
  // makes none.
  for (int i = threadIdx.x; i < (BM - p.tokens * G) * 8 * DB * STAGES; i += C::THREADS) {
    const int block = i / ((BM - p.tokens * G) * 8), at = i - block * ((BM - p.tokens * G) * 8);
    *reinterpret_cast<uint4*>(q_s + block * (BM * 128) + p.tokens * G * 128 + at * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_async_smem();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_free[s], 256);
    }
    mbar_init(k_full, 1);
    *s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"((uint64_t)&p.kv_map) : "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"((uint64_t)&p.q_map) : "memory");
  }
  if (warp == 1) tmem_alloc(tmem_slot, C::TMEM_COLS);
  const int n_tiles = __shfl_sync(0xffffffffu, max(0, end - begin), 0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp == 0) {
    if (n_tiles > 0)
      load_tile<DB, BM>(k_s, p, BoxWalk<BM>(p, seq, key0, total, lane).row(p, kvh), 0, k_full, lane);
    if (n_tiles > 0) {
      bool ok = true;
      int sent = 0;
      const int token = __shfl_sync(0xffffffffu, first + begin * p.tokens, 0);
      for (int i = 0; i < n_tiles && ok; ++i) {
        const int st = i % STAGES;
        if (i >= STAGES) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], (uint32_t)(i / STAGES - 1) & 1, 11));
        if (!ok) break;
        if (elect_one()) load_rows<DB>(q_s + st * C::STAGE, p, token + i * p.tokens, kvh, G, &full[st]);
        __syncwarp();
        sent = i + 1;
      }
      if (!ok && lane == 0) {
        *s_abort = 1;
        mbar_wait(k_full, 0, 12);
        for (int i = max(0, sent - STAGES); i < sent; ++i) mbar_wait(&full[i % STAGES], (uint32_t)(i / STAGES) & 1, 12);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (n_tiles > 0) {
      const uint32_t idesc = instr_desc(BM, C::BN, false);
      const uint64_t k_desc = smem_desc(smem_u32(k_s), 16, 1024), q_desc = smem_desc(smem_u32(q_s), 16, 1024);
      bool ok = __all_sync(0xffffffffu, mbar_wait(k_full, 0, 13));
      for (int i = 0; i < n_tiles && ok; ++i) {
        const int st = i % STAGES, buf = i & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&full[st], (uint32_t)(i / STAGES) & 1, 14));
        if (ok && i >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&s_free[buf], (uint32_t)(i / 2 - 1) & 1, 15));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t qd = q_desc + (uint64_t)(st * (C::STAGE >> 4));
#pragma unroll
          for (int kk = 0; kk < DB * 4; ++kk)
            tc_mma(tmem_base + buf * C::BN, k_desc + (uint64_t)(((kk >> 2) * (BM * 128) + (kk & 3) * 32) >> 4),
                   qd + (uint64_t)(((kk >> 2) * (C::BN * 128) + (kk & 3) * 32) >> 4), idesc, kk > 0 ? 1u : 0u);
          tc_commit(&empty[st]);
          tc_commit(&s_full[buf]);
        }
        __syncwarp();
      }
      if (!ok) *s_abort = 1;
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ two threads per key, for half of the columns each
    const int quarter = warp & 3, half = (warp - 2) >> 2, at = quarter * 32 + lane, key = key0 + at;
    const bool counts = !CAP || (key < total && key_row(a, seq, key, kvh, 0) >= 0);
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const float* lse = a.lse + ((size_t)kvh * a.n_tokens + first) * G;
    const int rows = n * G, tile_rows = p.tokens * G;
    auto lse_of = [&](int i) {                          // of the tile's row `at`
      const int r = (begin + i) * tile_rows + at;
      return i < n_tiles && at < tile_rows && r < rows ? lse[r] : INFINITY;
    };
    const f32x2 scale2 = f2_pack(p.scale_log2, p.scale_log2);
    float next = half == 0 ? lse_of(0) : 0.f, sum = 0.f;
    bool ok = true;
    for (int i = 0; i < n_tiles; ++i) {
      const int buf = i & 1, t_first = (begin + i) * p.tokens;
      if (half == 0) {
        s_lse[buf * 128 + at] = -next;
        next = lse_of(i + 1);
      }
      pair_sync(1);                                     // all come here in every round, also behind a wait that ran out
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&s_full[buf], (uint32_t)(i / 2) & 1, 16));
      if (!ok) continue;
      tc_fence_after();
      uint32_t s[2][32];
      tmem_ld32_nowait(s[0], lane_addr + buf * C::BN + half * 64);
      tmem_ld32_nowait(s[1], lane_addr + buf * C::BN + half * 64 + 32);
      tmem_ld_wait();
      tc_fence_before();
      mbar_arrive(&s_free[buf]);
      // the rows of zeros: a key that is not finite gives no number there; under a cap those of the next request too, which are none of
      // this one's business
      const int own = (CAP ? min(tile_rows, rows - (begin + i) * tile_rows) : tile_rows) - half * 64;
      if (CAP ? own < 64 : half == 1 && tile_rows < BM) {
#pragma unroll
        for (int k = 0; k < 64; k += 8) {
          if (k + 8 <= own) continue;
#pragma unroll
          for (int e = 0; e < 8; ++e) s[k >> 5][(k & 31) + e] = k + e >= own ? 0u : s[k >> 5][(k & 31) + e];
        }
      }
      if (CAP) {
        cap32(s[0], p.cap, counts);
        cap32(s[1], p.cap, counts);
      }
      // rows behind the request's last and those that do not see every key of the tile
      const bool masked = key0 + BM - 1 > total - n + t_first || (begin + i + 1) * tile_rows > rows;
      const float4* ls = reinterpret_cast<const float4*>(s_lse + buf * 128 + half * 64);
      f32x2 w[4] = {0ull, 0ull, 0ull, 0ull};
      if (!masked) {
#pragma unroll
        for (int k = 0; k < 64; k += 4) {
          const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(ls + (k >> 2));
          float x0, x1, x2, x3;
          f2_unpack(f2_fma(f2_pack(__uint_as_float(s[k >> 5][k & 31]), __uint_as_float(s[k >> 5][(k & 31) + 1])), scale2, v.x), x0, x1);
          f2_unpack(f2_fma(f2_pack(__uint_as_float(s[k >> 5][(k & 31) + 2]), __uint_as_float(s[k >> 5][(k & 31) + 3])), scale2, v.y), x2, x3);
          w[(k >> 1) & 3] = f2_add(w[(k >> 1) & 3], f2_pack(scored_exp2(x0), scored_exp2(x1)));
          w[((k >> 1) + 1) & 3] = f2_add(w[((k >> 1) + 1) & 3], f2_pack(scored_exp2(x2), scored_exp2(x3)));
        }
      } else {
        // the first column that sees this key, and the first behind the rows
        const int lo = (key - (total - n) - t_first) * G - half * 64, hi = CAP ? own : min(tile_rows, rows - (begin + i) * tile_rows) - half * 64;
        const float* lf = reinterpret_cast<const float*>(ls);
        float x = 0.f;
#pragma unroll
        for (int k = 0; k < 64; ++k) {
          const float e = scored_exp2(fmaf(__uint_as_float(s[k >> 5][k & 31]), p.scale_log2, lf[k]));
          x += k >= lo && k < hi ? e : 0.f;
        }
        w[0] = f2_pack(x, 0.f);
      }
      sum += f2_sum(f2_add(w[0], w[1]), f2_add(w[2], w[3]));
    }
    if (!ok) *s_abort = 1;
    if (half == 1) s_part[at] = sum;
    pair_sync(1);
    if (ok && half == 0 && key < total) {
      sum += s_part[at];
      if (p.parts.chunks == 1) store_weight(a, seq, first, kvh, key, key - (total - n), sum);
      else if (n_tiles > 0) p.parts.w[(((size_t)seq * a.nkv + kvh) * p.parts.chunks + chunk) * p.parts.keys + key] = sum;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

bool make_q_map(CUtensorMap* map, const ScoredArgs& a, int tokens) {
  const long long dims[3] = {a.d, a.nq, a.n_tokens}, strides[3] = {2, (long long)a.d * 2, (long long)a.q_stride * 2};
  const int box[3] = {64, a.nq / a.nkv, tokens};
  return nhv_make_map_bf16_nd(map, a.q, 3, dims, strides, box);
}

int divisor(int a, int b) { return b == 0 ? a : divisor(b, a % b); }

template <int DB, bool CAP>
int launch_long(const LongArgs& p, int row_tiles, cudaStream_t stream) {
  static std::atomic<uint64_t> rows_done{0}, keys_done{0};
  const ScoredArgs& a = p.a;
  NHV_CUDA(nhv_allow_smem((const void*)scored_rows_tcgen05_kernel<DB, CAP>, Rows<DB>::SMEM, rows_done), "scored attention (tcgen05)");
  NHV_CUDA(nhv_allow_smem((const void*)scored_keys_tcgen05_kernel<DB, CAP>, Keys<DB>::SMEM, keys_done), "scored attention (tcgen05)");
  NHV_CUDA(nhv_launch(scored_rows_tcgen05_kernel<DB, CAP>, dim3(a.nkv, row_tiles, p.parts.splits), Rows<DB>::THREADS, Rows<DB>::SMEM, stream, p),
           "scored attention (tcgen05)");
  int rc = scored_join_rows(NHV_BF16, a, p.parts, stream);
  if (rc) return rc;
  NHV_CUDA(nhv_launch(scored_keys_tcgen05_kernel<DB, CAP>, dim3(a.nkv, p.key_tiles * p.parts.chunks, a.n_seqs), Keys<DB>::THREADS, Keys<DB>::SMEM, stream, p),
           "scored attention (tcgen05)");
  return scored_join_keys(a, p.parts, stream);
}

}  // namespace

NHV_API int nhv_scored_tcgen05_error() { return nhv_wait_error_take(); }
NHV_API void* nhv_scored_tcgen05_error_word() { return nhv_wait_error_address(); }

// Tiles of rows in the grid: at most one that is not full a request.
static long long long_row_tiles(int n_seqs, int n_tokens, int G, int d) { return (long long)n_tokens / ((d <= 128 ? 2 : 1) * (BM / G)) + n_seqs; }

bool scored_long_takes(int dtype, int nq, int nkv, int d, int page_size, int q_stride, float scale) {
  return scale > 0.f && dtype == NHV_BF16 && d % 8 == 0 && d <= SA_MAX_D && nq / nkv <= BM && page_size % 8 == 0 && q_stride > 0;
}

bool scored_long_reaches(const ScoredParts& p, int n_seqs, int n_tokens, int nq, int nkv, int d, int page_size, int n_pages) {
  const long long pool = (long long)n_pages * 2 * nkv * page_size, key_tiles = (long long)(p.keys / BM) * p.chunks;
  return pool < (1LL << 31) && key_tiles <= 65535 && long_row_tiles(n_seqs, n_tokens, nq / nkv, d) <= 65535;
}

size_t scored_long_plan(ScoredParts& p, int n_seqs, int n_tokens, int max_new, int max_keys, int nq, int nkv, int d) {
  const int G = nq / nkv, tokens = BM / G;
  p.tile_rows = tokens * G;
  p.tile_keys = BM;
  return scored_parts(p, n_seqs, n_tokens, max_new, max_keys, nq, nkv, d, (d <= 128 ? 2 : 1) * tokens * G, 64, 1400.0, SMS, 2 * SMS);
}

size_t scored_long_most(int n_seqs, int n_tokens, int max_keys, int nq, int nkv, int d) {
  const int G = nq / nkv;
  return scored_most_parts(n_seqs, n_tokens, max_keys, nq, nkv, d, BM / G * G, BM, 2 * SMS);
}

int scored_long_launch(ScoredArgs a, const ScoredParts& parts, cudaStream_t stream) {
  LongArgs p;
  p.a = a;
  p.cap = nhv_score_cap(a.scale, a.softcap);
  p.scale_log2 = a.softcap > 0.f ? 1.0f : a.scale * SA_LOG2E;
  p.parts = parts;
  p.tokens = BM / (a.nq / a.nkv);
  p.key_tiles = (int)(parts.keys / BM);
  const int db = (a.d + 63) / 64;
  p.box = divisor(a.page_size, 64);
  NHV_REQUIRE(nhv_make_map_bf16(&p.kv_map, a.pages, (long long)a.n_pages * 2 * a.nkv * a.page_size, a.d, a.d, 64, p.box),
              "scored attention (tcgen05): cannot encode the tensor map of the pool");
  NHV_REQUIRE(make_q_map(&p.q_map, a, p.tokens), "scored attention (tcgen05): cannot encode the tensor map of q");
  const long long row_tiles = long_row_tiles(a.n_seqs, a.n_tokens, a.nq / a.nkv, a.d);
  const bool cap = a.softcap > 0.f;
  switch (db) {
    case 1: return cap ? launch_long<1, true>(p, (int)row_tiles, stream) : launch_long<1, false>(p, (int)row_tiles, stream);
    case 2: return cap ? launch_long<2, true>(p, (int)row_tiles, stream) : launch_long<2, false>(p, (int)row_tiles, stream);
    case 3: return cap ? launch_long<3, true>(p, (int)row_tiles, stream) : launch_long<3, false>(p, (int)row_tiles, stream);
    default: return cap ? launch_long<4, true>(p, (int)row_tiles, stream) : launch_long<4, false>(p, (int)row_tiles, stream);
  }
}
