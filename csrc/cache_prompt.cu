// Attention of many new tokens over the 8-bit paged cache on the tensor cores (prompts, long turns).
//
// Row (token at position p, head h) sees the keys j < lim of its sequence: lim = p + 1, and where
// p lies inside the sequence's prefix, lim = prefix.
//     o = sum_j softmax_j(scale * q . k_j) v_j,   0 where no key is seen
//
// One block owns 256 rows of one key/value head, two tiles A and B of 128: the rows of a tile are the
// query heads of the group for 128 / group tokens, token first, so that a key is converted once for all
// of them.  Both products run on fp16 operands (tcgen05 kind::f16) with fp32 sums in tensor memory:
//
//   producer warp:  128 keys and values as bytes by TMA, page by page
//   convert warps:  bytes -> fp16, exact, into the operands' swizzled layout (two stages)
//   MMA warps:      one a row tile: S of 64 keys, two ahead of the softmax; then, for every P that
//                   comes, O += P V and the S after the next
//   softmax warps:  a thread has a row of 64 scores; P goes back into the first half of its S
//
// The scales, powers of two of 16 keys each, stay outside the products: a key block's multiplies its
// scores, a value block's enters the exponent, p = exp2(x + ev - M) with M the maximum of x + ev, so that
// p <= 2^8 (M lags by as much) is rounded to fp16 beside the largest product of weight and value scale; the
// sum of the weights takes each block's sum times 2^-ev in fp32.  Query rows are shifted by a power of two
// into fp16's range first: bf16 values keep all their bits down to 2^-27 of the row's largest.
//
// TMEM (512 columns): S_X0 and S_X1, 64 columns each, for tiles A and B, then O_A and O_B, 128 each; P is
// packed fp16 in the first 32 columns of its S and read from there as the A operand.  With one S of
// 128 keys a tile (the same columns), scores to P to products is a chain that leaves the tensor
// cores idle for more than half of the time; with two of 64 the next scores are there when a softmax ends.
// Measured on B200: five prompts to 4096 tokens (13703 in all), 16 and 4 heads, every token sees its whole
// prompt: 393 us by itself, 873 TFLOP/s of 1641, and 407 us, 844 TFLOP/s, between other work at the clocks that it
// leaves; tensor pipe active 39 % under the profiler (430 us there).  What
// bounds it: the products with next to nothing between them take 350 us, the softmax with half of the
// products 401 (both before the order of blocks below, 416).  One S of 128 keys a tile: 489 us; one MMA warp
// for both tiles: 478 us, since issuing takes as long as the products; a row's softmax on two warps: 473 us.
// O is rescaled only when a row's maximum grows by more than 2^8; only then is the last product
// waited for.  Registers: 512 threads start with 128 each; the softmax groups take 184, the converters
// keep 88 and the producer and MMA group 56 (the sum is the same).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "serving.h"

using namespace mimir;

namespace {

constexpr int kTile = 128;
constexpr int kHalf = 64;                               // keys of a turn
constexpr int kThreads = 512;
constexpr uint32_t kTileBytes = kTile * kCacheDim * 2;  // 32 KB of fp16
constexpr uint32_t kChunkBytes = kTileBytes / 2;        // one half of 64 dimensions
constexpr uint32_t kRawBytes = kTile * kCacheDim;       // 16 KB of bytes
constexpr float kRescaleThreshold = 8.f;
constexpr float kLowest = -3e38f;
constexpr int kScaleRing = 4;

struct __align__(8) Barriers {
  uint64_t q_full, q_ready;      // raw rows have come; they are fp16
  uint64_t raw_full[2];          // keys, values
  uint64_t raw_empty[2];
  uint64_t scales_full[kScaleRing];
  uint64_t k_full[2], v_full[2]; // converted
  uint64_t k_empty[2], v_empty[2];
  uint64_t s_full[2][2], p_full[2][2];  // per row tile and buffer
  uint64_t o_done[2][2];                // the same, of products
  uint64_t mma_done;
  uint32_t tmem_base;
  int pad;
};

constexpr uint32_t kSmemKV = 2 * kTileBytes;                 // stage s: K at +2s tiles, V at +2s+1
constexpr uint32_t kSmemRaw = 6 * kTileBytes;                // K bytes, V bytes
constexpr uint32_t kSmemScales = kSmemRaw + 2 * kRawBytes;   // [kScaleRing][8 blocks][k, v]
constexpr uint32_t kSmemBar = kSmemScales + kScaleRing * 16 * sizeof(float);
constexpr uint32_t kSmemBytes = kSmemBar + sizeof(Barriers);
static_assert(kSmemBytes <= 232448, "shared memory of a block");

__device__ __forceinline__ uint8_t* q_tile(uint8_t* b, int x) { return b + x * kTileBytes; }
__device__ __forceinline__ uint8_t* k_stage(uint8_t* b, int s) { return b + kSmemKV + 2 * s * kTileBytes; }
__device__ __forceinline__ uint8_t* v_stage(uint8_t* b, int s) { return k_stage(b, s) + kTileBytes; }
__device__ __forceinline__ uint8_t* raw_buffer(uint8_t* b, int kv) { return b + kSmemRaw + kv * kRawBytes; }

// Instruction descriptor: fp16 A and B, fp32 D.
__host__ __device__ constexpr uint32_t idesc_f16_f32(int M, int N, int b_mn) {
  return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// Issued by the lane for which `leader` holds; the whole warp goes through the code, so that operands stay
// in uniform registers.  D[tmem] (+)= A[smem] * B[smem], D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32_u(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
      "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]),
      "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]),
      "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::
          "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
template <int kRegs>
__device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {  // four bytes to fp16
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
// Two fp32 values in one register pair: products, sums and the like of both at once.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split_pair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
template <bool kBf16>
__device__ __forceinline__ float2 unpack(uint32_t w) {
  return kBf16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w)) : __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack(float a, float b) {
  return kBf16 ? pack_bf16x2(a, b) : half2_bits(a, b);
}

template <bool kBf16>
__global__ void __launch_bounds__(kThreads, 1)
    cache_prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_pages,
                        const AttentionParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];  // what the swizzle needs
  if (smem_u32(smem) & 1023) {
    if (threadIdx.x == 0) record_status(p.status, kCacheTimeout);
    return;
  }
  Barriers* bar = reinterpret_cast<Barriers*>(smem + kSmemBar);
  float* scale_ring = reinterpret_cast<float*>(smem + kSmemScales);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // uniform
  const int kvh = blockIdx.x % p.KV, group = p.group;
  const int tokens = kTile / group, per = 2 * tokens;  // tokens of a tile, and of this block

  after_previous();
  const int last = gridDim.x / p.KV - 1;
  int lo, tok0;  // this block's sequence (p.n: none) and first token in it
  if (p.n <= 32) {
    // Blocks of the longest sequences come first, within a sequence those of its last tokens, which see most where
    // it is causal: the GPU's last blocks are then short ones (five prompts of 1343 to 4096 tokens: 416 -> 392 us).
    // Lane i has sequence i.
    const int at = min(lane, p.n), slot = at < p.n ? p.seqs[at] : -1;
    const int keys = slot >= 0 && slot < p.slots ? p.lens[slot] : 0;
    const NewRows rows = at < p.n ? new_rows(p.cu, at, p.tokens) : NewRows{0, 0, true};
    const int blocks = (rows.count + per - 1) / per;
    int before = 0;
    for (int i = 0; i < p.n; ++i) {
      const int keys_i = __shfl_sync(0xffffffffu, keys, i), blocks_i = __shfl_sync(0xffffffffu, blocks, i);
      if (keys_i > keys || (keys_i == keys && i < lane)) before += blocks_i;
    }
    const int mine = before + blocks - 1 - (int)(blockIdx.x / p.KV);
    const uint32_t owner = __ballot_sync(0xffffffffu, mine >= 0 && mine < blocks);
    lo = owner != 0 ? __ffs(owner) - 1 : p.n;
    tok0 = __shfl_sync(0xffffffffu, mine, lo & 31) * per;
  } else {
    // Sequence i has at most new / per + 1 blocks: those from cu[i] / per + 2 i on are its own, and some stay
    // empty.  The last ones come first.
    const int b = last - blockIdx.x / p.KV;
    lo = 0;
    for (int size = p.n + 1; size > 1;) {
      const int step = (size + 31) / 32;
      const int at = min(lo + lane * step, p.n);
      const int c = __popc(__ballot_sync(0xffffffffu, lo + lane * step < lo + size && max(p.cu[at], 0) / per + 2 * at <= b));
      const int next = lo + max(c - 1, 0) * step;
      size = min(step, lo + size - next);
      lo = next;
    }
    if (b == last) lo = p.n;  // as it is where the bounds are right
    tok0 = lo < p.n ? (b - (max(p.cu[lo], 0) / per + 2 * lo)) * per : 0;
  }
  if (lo >= p.n) {
    // rows that belong to no sequence: one block per head, which has never any of its own, clears them,
    // and one looks at the bounds
    if (blockIdx.x / p.KV == (p.n <= 32 ? last : 0)) {
      auto clear_rows = [&](int from, int to) {
        uint4* o = reinterpret_cast<uint4*>(p.out);
        constexpr int kWords = kCacheDim * 2 / 16;
        for (int64_t x = threadIdx.x; x < (int64_t)(to - from) * group * kWords; x += kThreads) {
          const int64_t row = x / kWords;
          o[((from + row / group) * p.H + kvh * group + row % group) * kWords + x % kWords] = make_uint4(0, 0, 0, 0);
        }
      };
      if (p.first_batch) clear_rows(0, min(max(p.cu[0], 0), p.tokens));
      if (p.last_batch) clear_rows(min(max(p.cu[p.n], 0), p.tokens), p.tokens);
      if (kvh == 0) check_bounds(p.cu, p.n, p.tokens, p.status);
    }
    return;
  }
  const NewRows rows = new_rows(p.cu, lo, p.tokens);
  const int first_row = rows.first, count = rows.count;
  if (tok0 < 0 || tok0 >= count) return;  // block-uniform, before any allocation
  const int slot = p.seqs[lo], prefix = p.prefix != nullptr ? p.prefix[lo] : 0;
  int len = 0;
  if (slot < 0 || slot >= p.slots) {
    if (threadIdx.x == 0) record_status(p.status, kCacheBadSlot);
  } else {
    len = rows.good ? p.lens[slot] : 0;
    if (threadIdx.x == 0 && len < count) record_status(p.status, kCacheBadLength);
    if (len > p.width * p.page) {
      len = p.width * p.page;
      if (threadIdx.x == 0) record_status(p.status, kCacheBadPage);
    }
    len = max(len, 0);
  }
  auto limit_of = [&](int tok) {  // keys that a token sees; it does not fall from token to token
    const int pos = len - count + tok;
    int lim = pos + 1;
    if (pos < prefix) lim = max(lim, prefix);
    return max(min(lim, len), 0);
  };
  const bool has_b = tok0 + tokens < count;
  // turns of 64 keys that each tile needs, and tiles of 128 keys
  const int turns_a = (limit_of(min(tok0 + tokens, count) - 1) + kHalf - 1) / kHalf;
  const int turns_b = has_b ? (limit_of(min(tok0 + per, count) - 1) + kHalf - 1) / kHalf : 0;
  const int turns = max(turns_a, turns_b), nkv = (turns + 1) / 2;

  if (threadIdx.x == 0) {
    mbar_init(&bar->q_full, 1);
    mbar_init(&bar->q_ready, 8);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bar->raw_full[s], 1);
      mbar_init(&bar->raw_empty[s], 4);
      mbar_init(&bar->k_full[s], 4);
      mbar_init(&bar->v_full[s], 4);
      mbar_init(&bar->k_empty[s], 2);
      mbar_init(&bar->v_empty[s], 2);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bar->s_full[s][i], 1);
        mbar_init(&bar->p_full[s][i], 4);
        mbar_init(&bar->o_done[s][i], 1);
      }
    }
    for (int s = 0; s < kScaleRing; ++s) mbar_init(&bar->scales_full[s], 16);
    mbar_init(&bar->mma_done, 2);
    fence_mbarrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&bar->tmem_base, 512);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_pages);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar->tmem_base;
  auto tS = [tmem](int x, int i) -> uint32_t { return tmem + x * 128 + (i & 1) * kHalf; };  // of turn i
  auto tO = [tmem](int x) -> uint32_t { return tmem + 256 + x * 128; };
  int* const status = p.status;

  if (warp < 4) {
    give_registers<56>();
    if (warp == 0) {
      // ------------------------------------------------------------ producer
      if (lane == 0) {
        const uint32_t box = tokens * group * 64 * 2;  // 64 dimensions of a tile's rows
        mbar_arrive_expect_tx(&bar->q_full, 2 * box * (has_b ? 2 : 1));
        for (int x = 0; x < (has_b ? 2 : 1); ++x)
          for (int half = 0; half < 2; ++half)
            tma_load_3d(smem_u32(q_tile(smem, x) + half * kChunkBytes), &map_q, &bar->q_full, half * 64, kvh * group,
                        first_row + tok0 + x * tokens);
      }
      __syncwarp();
      const int piece = min(p.page, kTile), pieces = kTile / piece;
      const int* row = p.table + (int64_t)max(slot, 0) * p.width;
      int base = -32, mine = 0, issued = 0;
      for (int j = 0; j < nkv; ++j) {
        if (j * pieces + pieces > base + 32) {  // page ids of the pieces base .. base + 31, one a lane
          base = j * pieces;
          const int64_t tok = (int64_t)(base + lane) * piece;
          mine = 0;
          if (tok < len) {
            mine = row[tok >> p.page_shift];
            if (mine < 0 || mine >= p.npages) {
              record_status(status, kCacheBadPage);
              mine = 0;  // some page of the pool: the result is reported as wrong, the access is not
            }
          }
        }
        // Scales: lane 2y + kv has block y's.  The ring's slot was read for tile j - 4, before the second
        // scores of tile j - 3, and those before the keys of tile j - 1 were converted.
        if (j > 0 && !warp_wait(&bar->raw_empty[0], (j - 1) & 1, status, kCacheTimeout)) break;
        const int y = lane >> 1;
        const int tok_y = j * kTile + (y & 7) * kCacheBlock;
        const int page_y = __shfl_sync(0xffffffffu, mine, (tok_y / piece - base) & 31);
        if (lane < 16) {
          const float* src = p.scales + (((int64_t)page_y * 2 + (lane & 1)) * p.KV + kvh) * (p.page / kCacheBlock) +
                             (tok_y & (p.page - 1)) / kCacheBlock;
          const uint32_t dst = smem_u32(scale_ring + (j % kScaleRing) * 16 + lane);
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(tok_y < len ? 4 : 0) : "memory");
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&bar->scales_full[j % kScaleRing])) : "memory");
        }
        const int here = min(pieces, (len - j * kTile + piece - 1) / piece);
        bool ok = true;
        for (int kv = 0; kv < 2; ++kv) {
          if (kv == 1 && j > 0) ok = warp_wait(&bar->raw_empty[1], (j - 1) & 1, status, kCacheTimeout);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&bar->raw_full[kv], here * piece * kCacheDim);
          for (int x = 0; x < here; ++x) {
            const int page = __shfl_sync(0xffffffffu, mine, j * pieces + x - base);
            if (lane == 0)
              tma_load_3d(smem_u32(raw_buffer(smem, kv) + x * piece * kCacheDim), &map_pages, &bar->raw_full[kv], 0,
                          (j * kTile + x * piece) & (p.page - 1), (page * 2 + kv) * p.KV + kvh);
          }
          issued = 2 * j + kv + 1;
        }
        if (!ok) break;
      }
      // No copy into this block's shared memory may outlive it.
      asm volatile("cp.async.wait_all;" ::: "memory");
      warp_wait(&bar->q_full, 0, status, kCacheTimeout);
      for (int kv = 0; kv < 2; ++kv) {
        const int loads = (issued + 1 - kv) / 2;
        if (loads > 0) warp_wait(&bar->raw_full[kv], (loads - 1) & 1, status, kCacheTimeout);
      }
    } else if (warp < 3) {
      // ------------------------------------------------------------ MMA issuer of tile x
      const uint32_t idesc_qk = idesc_f16_f32(128, kHalf, 0);
      const uint32_t idesc_pv = idesc_f16_f32(128, 128, 1);
      const uint32_t leader = elect_one_sync();
      const int x = warp - 1, mine = x == 0 ? turns_a : turns_b;
      auto commit = [&](uint64_t* b) {
        if (leader) mma_commit(b);
      };
      // Descriptors: the address field counts 16 bytes, and no sum of offsets leaves it.
      const uint64_t dq = smem_desc(smem_u32(smem), 16, 1024, kLayoutSW128);
      const uint64_t dk = smem_desc(smem_u32(smem + kSmemKV), 16, 1024, kLayoutSW128);
      const uint64_t dv = smem_desc(smem_u32(smem + kSmemKV + kTileBytes), kChunkBytes, 1024, kLayoutSW128);
      auto issue_s = [&](int i) {  // keys 64 i .. 64 i + 63
        const uint64_t a = dq + x * (kTileBytes >> 4), b = dk + (i >> 1 & 1) * (2 * kTileBytes >> 4) + (i & 1) * (kHalf * 128 >> 4);
        const uint32_t d = tS(x, i);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t off = ((k >> 2) * kChunkBytes + (k & 3) * 32) >> 4;
          mma_ss(d, a + off, b + off, idesc_qk, k > 0 ? 1u : 0u, leader);
        }
        commit(&bar->s_full[x][i & 1]);
      };
      auto issue_pv = [&](int i) {
        const uint64_t b = dv + (i >> 1 & 1) * (2 * kTileBytes >> 4) + (i & 1) * (kHalf * 128 >> 4);
        const uint32_t d = tO(x), a = tS(x, i);
#pragma unroll
        for (int k = 0; k < 4; ++k)  // 16 keys: 8 packed columns of P, 2 KB of V
          mma_ts(d, a + k * 8, b + k * (2048 >> 4), idesc_pv, (i > 0 || k > 0) ? 1u : 0u, leader);
        commit(&bar->o_done[x][i & 1]);
      };
      int k_seen = -1, v_seen = -1;  // tiles whose keys and values are known to have come
      auto keys_ready = [&](int tile) {
        if (tile > k_seen && !warp_wait(&bar->k_full[tile & 1], (tile >> 1) & 1, status, kCacheTimeout)) return false;
        k_seen = tile;
        tc_fence_after();
        return true;
      };
      auto values_ready = [&](int tile) {
        if (tile > v_seen && !warp_wait(&bar->v_full[tile & 1], (tile >> 1) & 1, status, kCacheTimeout)) return false;
        v_seen = tile;
        return true;
      };
      // Both warps give every stage back after it has come, used or not, so that neither is a round ahead.
      bool ok = nkv > 0 && warp_wait(&bar->q_ready, 0, status, kCacheTimeout) && keys_ready(0);
      for (int i = 0; ok && i < min(2, mine); ++i) issue_s(i);
      if (ok) commit(&bar->k_empty[0]);
      for (int i = 0; ok && i < turns; ++i) {
        if (i < mine) ok = warp_wait(&bar->p_full[x][i & 1], (i >> 1) & 1, status, kCacheTimeout);
        if (!ok || !values_ready(i >> 1)) break;
        tc_fence_after();
        if (i < mine) issue_pv(i);
        if ((i & 1) || i == turns - 1) commit(&bar->v_empty[i >> 1 & 1]);
        if (i + 2 >= turns) continue;
        if (!keys_ready((i + 2) >> 1)) break;
        if (i + 2 < mine) issue_s(i + 2);
        if ((i & 1) || i + 2 == turns - 1) commit(&bar->k_empty[(i + 2) >> 1 & 1]);
      }
      // Every MMA that this warp issued completes before TMEM is released.
      commit(&bar->mma_done);
      warp_wait(&bar->mma_done, 0, status, kCacheTimeout);
    }
  } else if (warp >= 12) {
    // -------------------------------------------------------------- converters
    give_registers<88>();
    const int w = warp - 12, r0 = lane & 7, ch0 = lane >> 3;
    for (int j = 0; j < nkv; ++j) {
      const int s = j & 1;
      bool ok = true;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        if (j >= 2) ok = warp_wait(kv ? &bar->v_empty[s] : &bar->k_empty[s], ((j >> 1) - 1) & 1, status, kCacheTimeout);
        if (ok) ok = warp_wait(&bar->raw_full[kv], j & 1, status, kCacheTimeout);
        if (!ok) break;
        const uint32_t src = smem_u32(raw_buffer(smem, kv));
        const uint32_t dst = smem_u32(kv ? v_stage(smem, s) : k_stage(smem, s));
        const int stop = kv ? len - j * kTile : kTile;  // values beyond the sequence: any byte, NaN among them
        // eight rows times four 16-byte chunks at a time: no bank conflicts on either side
        uint4 in[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = w * 32 + (i >> 1) * 8 + r0, ch = ch0 + (i & 1) * 4;
          in[i] = lds128(src + r * 128 + ((ch ^ (r & 7)) << 4));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = w * 32 + (i >> 1) * 8 + r0, ch = ch0 + (i & 1) * 4;
          if (r >= stop) in[i] = make_uint4(0, 0, 0, 0);
          uint32_t o[8];
          widen(in[i].x, o[0], o[1]);
          widen(in[i].y, o[2], o[3]);
          widen(in[i].z, o[4], o[5]);
          widen(in[i].w, o[6], o[7]);
          const uint32_t to = dst + (ch >> 2) * kChunkBytes + r * 128;
          const int c2 = (ch & 3) * 2;
          st_shared_v4(to + ((c2 ^ (r & 7)) << 4), o[0], o[1], o[2], o[3]);
          st_shared_v4(to + (((c2 + 1) ^ (r & 7)) << 4), o[4], o[5], o[6], o[7]);
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bar->raw_empty[kv]);
          mbar_arrive(kv ? &bar->v_full[s] : &bar->k_full[s]);
        }
      }
      if (!ok) break;
    }
  } else {
    // -------------------------------------------------------------- softmax + epilogue of tile x
    take_registers<184>();
    const int x = (warp - 4) >> 2, wq = warp & 3, r = wq * 32 + lane;
    const int tok = tok0 + x * tokens + r / group, my_turns = x == 0 ? turns_a : turns_b;
    const bool valid = r < tokens * group && tok < count;
    const int lim = limit_of(min(tok, count - 1));
    const int min_lim = limit_of(min(tok0 + x * tokens, count - 1));
    const uint32_t lane_off = (uint32_t)(wq * 32) << 16;
    bool ok = warp_wait(&bar->q_full, 0, status, kCacheTimeout);
    // ---- this thread's query row to fp16, its largest value to [2^13, 2^14)
    float factor = 0.f;
    {
      const uint32_t row = smem_u32(q_tile(smem, x)) + r * 128;
      float top = 0.f;
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const uint4 v = lds128(row + (c >> 3) * kChunkBytes + (((c & 7) ^ (r & 7)) << 4));
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack<kBf16>(u[i]);
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      const int shift = max(min(13 - ((__float_as_int(top) >> 23) - 127), 120), -115);
      const float f = __int_as_float((shift + 127) << 23);
      factor = p.scale_log2 * __int_as_float((127 - shift) << 23);
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const uint32_t at = row + (c >> 3) * kChunkBytes + (((c & 7) ^ (r & 7)) << 4);
        const uint4 v = lds128(at);
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&v);
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 e = unpack<kBf16>(u[i]);
          o[i] = half2_bits(e.x * f, e.y * f);
        }
        st_shared_v4(at, o[0], o[1], o[2], o[3]);
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->q_ready);
    }
    float M = kLowest, l = 0.f;
    for (int i = 0; i < my_turns; ++i) {
      const int j = i >> 1;
      if (ok) ok = warp_wait(&bar->scales_full[j % kScaleRing], (j / kScaleRing) & 1, status, kCacheTimeout);
      if (ok) ok = warp_wait(&bar->s_full[x][i & 1], (i >> 1) & 1, status, kCacheTimeout);
      if (!ok) break;
      tc_fence_after();
      float sv[kHalf];
      {
        uint32_t raw[2][32];
#pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld32_nowait(tS(x, i) + lane_off + c * 32, raw[c]);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e) sv[c * 32 + e] = __uint_as_float(raw[c][e]);
      }
      const int rel = lim - i * kHalf;  // columns below it are seen
      const float4* sc = reinterpret_cast<const float4*>(scale_ring + (j % kScaleRing) * 16 + (i & 1) * 8);
      float alpha = 1.f;
      bool rescale = false;
      uint32_t pk[32];
      // Tiles that some row sees only in part are masked; the others do without those instructions.
      auto probabilities = [&](auto masked) {
        constexpr bool kMasked = decltype(masked)::value;
        if (kMasked) {
#pragma unroll
          for (int c = 0; c < kHalf; ++c) sv[c] = c >= rel ? -INFINITY : sv[c];
        }
        float mult[4], ev[4], inv[4];  // of the blocks: the scores' factor, log2 of the values' scale, its inverse
#pragma unroll
        for (int y = 0; y < 4; y += 2) {
          const float4 two = sc[y / 2];
          mult[y] = factor * two.x, mult[y + 1] = factor * two.z;
          // NaN stays NaN
          ev[y] = two.y == two.y ? (float)((__float_as_int(two.y) >> 23) - 127) : two.y;
          ev[y + 1] = two.w == two.w ? (float)((__float_as_int(two.w) >> 23) - 127) : two.w;
          inv[y] = two.y == two.y ? __int_as_float(0x7f000000 - __float_as_int(two.y)) : two.y;
          inv[y + 1] = two.w == two.w ? __int_as_float(0x7f000000 - __float_as_int(two.w)) : two.w;
        }
        float mx = kLowest;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float* v = sv + y * 16;
          const float t0 = max3(v[0], v[1], v[2]), t1 = max3(v[3], v[4], v[5]), t2 = max3(v[6], v[7], v[8]);
          const float t3 = max3(v[9], v[10], v[11]), t4 = max3(v[12], v[13], v[14]);
          mx = fmaxf(mx, fmaf(max3(max3(t0, t1, t2), max3(t3, t4, v[15]), t0), mult[y], ev[y]));
        }
        if (mx > M + kRescaleThreshold) {
          alpha = fast_exp2(M - mx);
          rescale = i > 0;
          M = mx;
        }
        l *= alpha;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const uint64_t m2 = pair_of(mult[y], mult[y]), a2 = pair_of(ev[y] - M, ev[y] - M);
          float sA = 0.f, sB = 0.f;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const int col = y * 16 + 2 * c;
            float a, d;
            split_pair(fma_pair(pair_of(sv[col], sv[col + 1]), m2, a2), a, d);
            a = fast_exp2(a), d = fast_exp2(d);
            if (kMasked) {  // also beside a poisoned block's NaN
              if (col >= rel) a = 0.f;
              if (col + 1 >= rel) d = 0.f;
            }
            sA += a; sB += d;
            pk[y * 8 + c] = half2_bits(a, d);
          }
          const float both = sA + sB;
          if (!kMasked || both != 0.f) l = fmaf(both, inv[y], l);  // a block that is not seen adds nothing
        }
      };
      if ((i + 1) * kHalf > min_lim) probabilities(std::true_type{});
      else probabilities(std::false_type{});
      if (__any_sync(0xffffffff, rescale)) {  // O is touched: its last product has to be done
        ok = warp_wait(&bar->o_done[x][(i - 1) & 1], (i - 1) >> 1 & 1, status, kCacheTimeout);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float ov[32];
          tmem_ld32(tO(x) + lane_off + c * 32, ov);
#pragma unroll
          for (int e = 0; e < 32; ++e) ov[e] *= alpha;
          tmem_st32(tO(x) + lane_off + c * 32, ov);
        }
      }
      tmem_st32_u(tS(x, i) + lane_off, pk);  // over scores that have been loaded
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->p_full[x][i & 1]);
    }
    // A parity tells only neighbouring phases apart.  Of the last two products either may be done by now, so they have
    // a barrier each (with one for both, the wait for the first would miss its phase when the second is done too); all
    // before them were done when the last scores came.
    for (int i = max(my_turns - 2, 0); ok && i < my_turns; ++i)
      ok = warp_wait(&bar->o_done[x][i & 1], i >> 1 & 1, status, kCacheTimeout);
    tc_fence_after();
    const float inv_l = l > 0.f || l != l ? 1.f / l : 0.f;
    uint4* dst = reinterpret_cast<uint4*>(p.out) + ((int64_t)(first_row + tok) * p.H + kvh * group + r % group) * (kCacheDim / 8);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float ov[32];
      if (ok && my_turns > 0) {
        tmem_ld32(tO(x) + lane_off + c * 32, ov);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) ov[i] = 0.f;
      }
      if (valid) {
#pragma unroll
        for (int v = 0; v < 4; ++v)
          dst[c * 4 + v] = make_uint4(pack<kBf16>(ov[v * 8] * inv_l, ov[v * 8 + 1] * inv_l), pack<kBf16>(ov[v * 8 + 2] * inv_l, ov[v * 8 + 3] * inv_l),
                                      pack<kBf16>(ov[v * 8 + 4] * inv_l, ov[v * 8 + 5] * inv_l), pack<kBf16>(ov[v * 8 + 6] * inv_l, ov[v * 8 + 7] * inv_l));
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <bool kBf16>
cudaError_t launch(const CUtensorMap& map_q, const CUtensorMap& map_pages, const AttentionParams& p, cudaStream_t stream) {
  static bool set[64] = {false};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (!set[dev]) {
    err = cudaFuncSetAttribute(cache_prompt_kernel<kBf16>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (err != cudaSuccess) return err;
    set[dev] = true;
  }
  const int per = 2 * (kTile / p.group);
  const int64_t grid = (int64_t)p.KV * (p.tokens / per + 2 * p.n + 1);
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  return launch_after_previous(cache_prompt_kernel<kBf16>, dim3((unsigned)grid), kThreads, kSmemBytes, stream, map_q, map_pages, p);
}

}  // namespace

namespace mimir {
cudaError_t launch_cache_prompt(const CUtensorMap& map_q, const CUtensorMap& map_pages, const AttentionParams& p, bool bf16,
                                cudaStream_t stream) {
  return bf16 ? launch<true>(map_q, map_pages, p, stream) : launch<false>(map_q, map_pages, p, stream);
}
}  // namespace mimir
