// Attention of new tokens over the 8-bit paged cache, split along the keys (few rows a sequence).
//
// Row (token at position p, head h) sees the keys j < lim of its sequence: lim = p + 1, and where
// p lies inside the sequence's prefix, lim = prefix.
//     o = sum_j softmax_j(scale * q . k_j) v_j,   0 where no key is seen
//
// The time of a decoding step is that of reading the cache once, so the kernel is built around the
// bytes.  All (sequence, key/value head, tile of 16 rows) segments, cut into units of 64 keys, form
// one line that is dealt to the grid's blocks in equal shares: a long sequence is spread over many
// blocks and short ones share a block.  A row tile holds the query heads of the group times the
// tokens, so that a key is read once for all of them.  A producer warp brings 64 keys and values
// (8 KB each) a stage by TMA with the 128-byte swizzle; four warps take 16 keys each, with a
// softmax of their own, and join at the end of a segment.  A segment that spans blocks leaves partial
// sums, and the last of its blocks to finish joins them in the order of the keys (so that results do
// not depend on which block that is).
//
// Matrix products are m16n8k16 with fp16 operands and fp32 sums, keys or head dimensions as the 16 and
// query rows as the 8 columns: a group's few rows fill the narrow side.  Bytes become fp16
// exactly; the scales, powers of two, stay outside: a key block's multiplies its scores, a value
// block's enters the exponent of the probability that multiplies the values, exp2(x + ev - M) with a
// maximum M of x + ev of its own, beside exp2(x - m) for the sum.  Probabilities are rounded to fp16 for the
// product: to 11 bits, and below 2^-14 to 2^-25 of the largest product of weight and value scale.  Query rows are
// shifted by a power of two into fp16's range: bf16 values keep all their bits down to 2^-27 of the row's largest,
// smaller ones are rounded to 2^-38 of it.
// The contraction over the head dimension may run in any order: thread c of a quad takes the bytes
// 32c..32c+31 of a key row, which two 16-byte loads bring without bank conflicts under the swizzle, and
// the same dimensions of the query rows.  Of the values thread (g, c) takes the bytes 16g..16g+15 of
// four rows; row g of product j is dimension 16g + 2j, row g + 8 the one after it.
//
// Measured on B200 (16 query and 4 key/value heads, one new token): 64 sequences to 8000 tokens 41 us for
// 166 MB; 8 sequences to 100001 tokens 75 us for 391 MB (5.2 TB/s; 6.4 TB/s between two lengths, where the
// some 10 us of start and joining cancel); DRAM reads are the cache's bytes and no more.  24 sequences to
// 2100 tokens, 7 tokens, 20 and 20 heads: 44 us for 138 MB.  With the rows as the wide side of the products
// (half of it empty) a warp needs 406 instructions for 16 keys instead of some 200: 55, 87 and 83 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "serving.h"

using namespace mimir;

namespace {

constexpr int kKeys = kAttentionKeys;          // keys of a unit
constexpr int kWarps = 4;                      // consumers
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kRows = kAttentionRows;          // rows of a full tile
constexpr uint32_t kHalfStage = kKeys * kCacheDim;
constexpr uint32_t kStageBytes = 2 * kHalfStage;
constexpr int kOutLd = 132;                    // floats of a row in the join buffer
constexpr int kQueryLd = 272;                  // bytes of a query row in shared memory: 16 spread over the banks
constexpr int kWindow = 32;                    // sequences whose lengths a block keeps at hand
constexpr float kLowest = -3e38f;
constexpr float kGrowth = 8.f;                 // maxima move only when they grow by more than 2^8
constexpr int kEnds = kAttentionEnds;

using Params = AttentionParams;

// kTiles: products' widths of 8 that make a row tile.  Eight rows leave registers and shared memory for three
// blocks an SM, sixteen for two.  Either takes any number of rows a sequence: what the host believes of it
// decides only which is faster.
template <int kTiles>
struct Shape {
  static constexpr int kRowsHeld = 8 * kTiles;
  static constexpr int kStages = kTiles == 1 ? 3 : 4;
  static constexpr int kBlocksPerSm = kTiles == 1 ? 3 : 2;
};

template <int kStages>
struct __align__(8) Barriers {
  uint64_t full[kStages];
  uint64_t empty[kStages];
  uint64_t q_full[2];
  uint64_t q_empty[2];
};

struct __align__(8) Seq {
  int len, row, count, slot, prefix, pad;  // tokens, first new row, new rows, page table row
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t f16_of_lo(uint32_t w) {  // bytes 0, 1 of w as two fp16
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t f16_of_hi(uint32_t w) {  // bytes 2, 3
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t w) {  // 16-bit values: row g, columns 2c, 2c + 1 a thread
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
  return r;
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
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::
          "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ float2 get(uint32_t w) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w)); }
  static __device__ __forceinline__ uint32_t put(float a, float b) { return pack_bf16x2(a, b); }
  static __device__ __forceinline__ __nv_bfloat16 one(float a) { return __float2bfloat16_rn(a); }
};
template <>
struct Pair<__half> {
  static __device__ __forceinline__ float2 get(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
  static __device__ __forceinline__ uint32_t put(float a, float b) { return half2_bits(a, b); }
  static __device__ __forceinline__ __half one(float a) { return __float2half_rn(a); }
};

// Keys that the row of token `tok` (of s.count new ones) sees.
__device__ __forceinline__ int row_limit(const Seq& s, int tok) {
  const int pos = s.len - s.count + tok;
  int lim = pos + 1;
  if (pos < s.prefix) lim = max(lim, s.prefix);
  return max(min(lim, s.len), 0);
}

// A part of a segment: tiles t0 .. t1 - 1 of sequence i, head h, row tile rt.
struct Segment {
  int i, h, rt, t0, t1, tiles;
  int64_t first_tile;  // where its tiles start on the line
};

// Sequence i of the batch; a bad slot or length is reported and read as no tokens.
__device__ Seq load_seq(const Params& p, int i) {
  Seq s;
  const NewRows rows = new_rows(p.cu, i, p.tokens);
  s.row = rows.first, s.count = rows.count;
  s.slot = p.seqs[i];
  s.prefix = p.prefix != nullptr ? p.prefix[i] : 0;
  s.len = 0;
  if (s.slot < 0 || s.slot >= p.slots) {
    s.slot = 0;
    if (s.count > 0) record_status(p.status, kCacheBadSlot);
  } else {
    s.len = rows.good ? p.lens[s.slot] : 0;
    if (s.len < s.count || !rows.good) record_status(p.status, kCacheBadLength);
    if (s.len < 0) s.len = 0;
    if (s.len > p.width * p.page) {
      s.len = p.width * p.page;
      record_status(p.status, kCacheBadPage);
    }
  }
  return s;
}
__device__ __forceinline__ int seq_tiles(const Seq& s) { return max((s.len + kKeys - 1) / kKeys, 1); }
template <int kMine>  // rows of a tile
__device__ __forceinline__ int seq_row_tiles(const Params& p, const Seq& s) {
  return (s.count * p.group + kMine - 1) / kMine;
}
template <int kMine>
__device__ __forceinline__ int64_t seq_units(const Params& p, const Seq& s) {
  return (int64_t)p.KV * seq_row_tiles<kMine>(p, s) * (seq_tiles(s) + kEnds);
}

// A block's share of the line, one segment at a time.
template <int kMine>
struct Walk {
  const Params& p;
  const Seq* window;   // sequences from `from` on: what a block's share meets, as a rule
  int from, i;         // i: the sequence at u, which starts at `base`
  int64_t base, u, end;
  Seq s;
  __device__ Seq seq(int x) const { return x - from < kWindow ? window[x - from] : load_seq(p, x); }
  __device__ bool next(Segment& g) {
    while (u < end) {
      int64_t units;
      while (base + (units = seq_units<kMine>(p, s)) <= u) {
        base += units;
        s = seq(++i);
      }
      const int rts = seq_row_tiles<kMine>(p, s);
      g.i = i;
      g.tiles = seq_tiles(s);
      const int length = g.tiles + kEnds;
      const int64_t local = u - base;
      int off;
      if (local >> 32) {
        const int64_t seg = local / length;
        off = (int)(local - seg * length);
        g.h = (int)(seg / rts);
        g.rt = (int)(seg % rts);
      } else {
        const uint32_t x = (uint32_t)local / (uint32_t)length;
        off = (int)((uint32_t)local - x * (uint32_t)length);
        g.h = (int)(x / (uint32_t)rts);
        g.rt = (int)(x % (uint32_t)rts);
      }
      const int stop = (int)min((int64_t)length, off + (end - u));
      g.first_tile = u - off + kEnds;
      g.t0 = max(off - kEnds, 0);
      g.t1 = max(stop - kEnds, 0);
      u += stop - off;
      if (g.t1 > g.t0) return true;
    }
    return false;
  }
};

// Joins the parts of a segment, blocks b0 .. b1: a warp a row, a lane four columns.
template <typename T, int kMine>
__device__ void join_parts(const Params& p, const Segment& sg, const Seq& s, int rows, int b0, int b1, int warp, int lane) {
  auto part_of = [&](int b) { return (int64_t)b * 2 + (b == b0 ? 1 : 0); };
  for (int r = warp; r < rows; r += kWarps) {
    float m = kLowest, sum = 0.f;
    for (int b = b0 + lane; b <= b1; b += 32) m = fmaxf(m, __ldcg(&p.part_ml[part_of(b) * kRows + r]).x);
    m = warp_max(m);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int base = b0; base <= b1; base += 32) {
      float w = 0.f;
      if (base + lane <= b1) {
        const float2 ml = __ldcg(&p.part_ml[part_of(base + lane) * kRows + r]);
        w = fast_exp2(ml.x - m);
        sum += ml.y * w;
      }
      const int here = min(32, b1 - base + 1);
#pragma unroll 8
      for (int j = 0; j < here; ++j) {
        const float f = __shfl_sync(0xffffffffu, w, j);
        const float4 x = __ldcg(reinterpret_cast<const float4*>(p.parts + (part_of(base + j) * kRows + r) * kCacheDim) + lane);
        o.x += x.x * f, o.y += x.y * f, o.z += x.z * f, o.w += x.w * f;
      }
    }
    sum = warp_sum(sum);
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    const int row = sg.rt * kMine + r;
    T* dst = reinterpret_cast<T*>(p.out) + ((int64_t)(s.row + row / p.group) * p.H + sg.h * p.group + row % p.group) * kCacheDim;
    reinterpret_cast<uint2*>(dst)[lane] = make_uint2(Pair<T>::put(o.x * inv, o.y * inv), Pair<T>::put(o.z * inv, o.w * inv));
  }
}

constexpr int kFewBlocks = 96;  // one sequence of 1000 keys: 84 blocks 10.5 us, 37 blocks 11.7

template <typename T, int kTiles>
__global__ void __launch_bounds__(kThreads, Shape<kTiles>::kBlocksPerSm) cache_attention_kernel(const __grid_constant__ CUtensorMap map, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int kMine = Shape<kTiles>::kRowsHeld;  // rows of a tile
  constexpr int kStages = Shape<kTiles>::kStages;
  float* joined = reinterpret_cast<float*>(smem + kStages * kStageBytes);        // [kWarps][kMine][kOutLd]
  float* stats = joined + kWarps * kMine * kOutLd;                               // [kWarps][kMine][4]: m, M, l
  float* block_scales = stats + kWarps * kMine * 4;                              // [kStages][4 blocks][k, v]
  uint8_t* query_base = reinterpret_cast<uint8_t*>(block_scales + kStages * 8);  // [2][kMine][kQueryLd]
  auto* bar = reinterpret_cast<Barriers<kStages>*>(query_base + 2 * kMine * kQueryLd);
  Seq* window = reinterpret_cast<Seq*>(bar + 1);                                 // [kWindow]
  // Units before a sequence, [n + 1]: needed until the join buffer is.  (Not in the stages: TMA writes those, in
  // no order with the ordinary stores of the line but by a proxy fence.)
  int64_t* first = reinterpret_cast<int64_t*>(joined);
  static_assert(sizeof(int64_t) * (kAttentionSeqs + 1) <= sizeof(float) * kWarps * kMine * kOutLd, "the line fits the join buffer");
  __shared__ int64_t scan_sums[kThreads / 32];
  __shared__ int64_t scan_base;
  __shared__ int last_of[2];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bar->full[s], 1 + 8);
      mbar_init(&bar->empty[s], kWarps);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bar->q_full[s], 32);
      mbar_init(&bar->q_empty[s], kWarps);
    }
    fence_mbarrier_init();
    tma_prefetch_desc(&map);
    scan_base = 0;
  }
  after_previous();
  // ---- the line of units
  for (int base = 0; base < p.n; base += kThreads) {
    const int i = base + (int)threadIdx.x;
    const int64_t units = i < p.n ? seq_units<kMine>(p, load_seq(p, i)) : 0;
    int64_t v = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += x;
    }
    if (lane == 31) scan_sums[warp] = v;
    __syncthreads();
    int64_t before = scan_base;
    for (int w = 0; w < warp; ++w) before += scan_sums[w];
    if (i < p.n) first[i] = before + v - units;
    __syncthreads();
    if (threadIdx.x == kThreads - 1) scan_base = before + v;
    __syncthreads();
  }
  if (threadIdx.x == 0) first[p.n] = scan_base;
  __syncthreads();
  const int64_t total = first[p.n];
  // Rows that belong to no sequence: a warp a block, when it has nothing else to do.
  auto clear_rows = [&]() {
    uint4* o = reinterpret_cast<uint4*>(p.out);
    const int64_t per = (int64_t)p.H * kCacheDim * sizeof(T) / 16, step = gridDim.x * 32;
    const int64_t before = p.first_batch ? min(p.cu[0], p.tokens) : 0;
    const int64_t after = p.last_batch ? min(max(p.cu[p.n], 0), p.tokens) : p.tokens;
    for (int64_t k = blockIdx.x * 32 + lane; k < before * per; k += step) o[k] = make_uint4(0, 0, 0, 0);
    for (int64_t k = after * per + blockIdx.x * 32 + lane; k < p.tokens * per; k += step) o[k] = make_uint4(0, 0, 0, 0);
  };
  // A unit takes about four times as long as joining a part does, and the last block of a segment joins all of its
  // parts: few long segments are shared by fewer blocks, so that units / blocks + parts / 4 is least, but by
  // kFewBlocks where there are units for them, and with whole units a block.  One sequence, 4 key/value heads, in
  // us, with all blocks and so: 6128 keys 20.4, 13.1; 24000 keys 25.3, 20.4; three of 6128 keys 21.9, 20.1.
  const int64_t best = max((int64_t)sqrtf((float)total * p.join_cost), (int64_t)kFewBlocks);
  int64_t blocks = min((int64_t)gridDim.x, total);
  if (best < blocks) {  // total < blocks^2 / 4 then
    const uint32_t each = (uint32_t)total / (uint32_t)best;
    blocks = min(blocks, (int64_t)(((uint32_t)total + each - 1) / each));
  }
  if (blockIdx.x >= blocks) {
    if (warp == kWarps) clear_rows();
    return;
  }
  auto share = [&](int64_t b) {
    return total < (1 << 22) ? (int64_t)((uint32_t)(total * b) / (uint32_t)blocks) : total * b / blocks;
  };
  Walk<kMine> walk{p, window, 0, 0, 0, share(blockIdx.x), share(blockIdx.x + 1), Seq{}};
  {
    int lo = 0, hi = p.n - 1;  // the last sequence with first <= u (empty ones have no units)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= walk.u) lo = mid;
      else hi = mid - 1;
    }
    walk.from = walk.i = lo;
    walk.base = first[lo];
  }
  if (threadIdx.x < kWindow && walk.from + (int)threadIdx.x < p.n) window[threadIdx.x] = load_seq(p, walk.from + threadIdx.x);
  __syncthreads();
  walk.s = window[0];
  const int piece = min(p.page, kKeys), pieces = kKeys / piece;  // keys that lie together, and their number in a unit

  // The tiles that a row tile needs: keys up to the largest limit of its rows.
  auto tiles_needed = [&](const Seq& s, int rt) {
    return (row_limit(s, min((rt * kMine + kMine - 1) / p.group, s.count - 1)) + kKeys - 1) / kKeys;
  };
  Segment sg;

  if (warp == kWarps) {
    // ------------------------------------------------------------ producer
    int it = 0;
    bool ok = true;
    for (int turn = 0; ok && walk.next(sg); ++turn) {
      const Seq& s = walk.s;
      // query rows of the tile, 16 bytes a lane, zeros beyond the last
      if (turn >= 2 && !warp_wait(&bar->q_empty[turn & 1], ((turn >> 1) - 1) & 1, p.status, kCacheTimeout)) break;
      for (int x = lane; x < kMine * 16; x += 32) {
        const int r = sg.rt * kMine + (x >> 4), tok = r / p.group;
        const bool held = tok < s.count;
        const T* src = reinterpret_cast<const T*>(p.q);
        if (held) src += (int64_t)(s.row + tok) * p.q_tok + (sg.h * p.group + r % p.group) * p.q_head + (x & 15) * 8;
        const uint32_t dst = smem_u32(query_base + ((turn & 1) * kMine + (x >> 4)) * kQueryLd + (x & 15) * 16);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(held ? 16 : 0) : "memory");
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&bar->q_full[turn & 1])) : "memory");
      const int t1 = min(sg.t1, tiles_needed(s, sg.rt));
      const int* row = p.table + (int64_t)s.slot * p.width;
      int base = -32, mine = -1;  // page ids of the pieces base .. base + 31, one a lane
      for (int t = sg.t0; ok && t < t1; ++t, ++it) {
        const int st = it % kStages;
        if (t * pieces + pieces > base + 32) {
          base = t * pieces;
          const int64_t tok = (int64_t)(base + lane) * piece;
          mine = 0;
          if (tok < s.len) {
            mine = row[tok >> p.page_shift];
            if (mine < 0 || mine >= p.npages) {
              record_status(p.status, kCacheBadPage);
              mine = 0;  // some page of the pool: the result is reported as wrong, the access is not
            }
          }
        }
        if (it >= kStages && !warp_wait(&bar->empty[st], ((it / kStages) - 1) & 1, p.status, kCacheTimeout)) {
          ok = false;
          break;
        }
        // scales: lane 2b of block b the keys', lane 2b + 1 the values'
        const int b = (lane >> 1) & 3;
        const int tok_b = t * kKeys + b * kCacheBlock;
        const int page_b = __shfl_sync(0xffffffffu, mine, (tok_b / piece - base) & 31);
        const float* src = p.scales + (((int64_t)page_b * 2 + (lane & 1)) * p.KV + sg.h) * (p.page / kCacheBlock) +
                           (tok_b & (p.page - 1)) / kCacheBlock;
        if (lane < 8) {
          const uint32_t dst = smem_u32(block_scales + st * 8 + lane);
          const int size = tok_b < s.len ? 4 : 0;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&bar->full[st])) : "memory");
        }
        const int here = min(pieces, (s.len - t * kKeys + piece - 1) / piece);
        if (lane == 0) mbar_arrive_expect_tx(&bar->full[st], here * piece * kCacheDim * 2);
        for (int x = 0; x < here; ++x) {
          const int page = __shfl_sync(0xffffffffu, mine, t * pieces + x - base);
          if (lane < 2) {  // lane 0 the keys, lane 1 the values
            const uint32_t dst = smem_u32(smem + st * kStageBytes + lane * kHalfStage + x * piece * kCacheDim);
            tma_load_3d(dst, &map, &bar->full[st], 0, (t * kKeys + x * piece) & (p.page - 1), (page * 2 + lane) * p.KV + sg.h);
          }
          __syncwarp();
        }
      }
    }
    // no copy into this block's shared memory may outlive it
    asm volatile("cp.async.wait_all;" ::: "memory");
    for (int j = max(0, it - kStages); j < it; ++j) warp_wait(&bar->full[j % kStages], (j / kStages) & 1, p.status, kCacheTimeout);
    clear_rows();
    return;
  }

  // -------------------------------------------------------------- consumers
  const int g = lane >> 2, c = lane & 3;
  int it = 0;
  bool ok = true;
  Segment split[2];
  int has_split = 0;
  auto block_of = [&](int64_t unit) { return (int)(((unit + 1) * blocks - 1) / total); };
  for (int turn = 0; walk.next(sg); ++turn) {
    const Segment cur = sg;
    if (ok) ok = warp_wait(&bar->q_full[turn & 1], (turn >> 1) & 1, p.status, kCacheTimeout);
    const Seq s = walk.s;
    const int t1 = min(cur.t1, tiles_needed(s, cur.rt));
    const int rows = min(s.count * p.group - cur.rt * kMine, kMine);
    // Rows 8n + g, dimensions 32c .. 32c + 31, as the products' second operand; and of rows
    // 8n + 2c and 8n + 2c + 1, whose scores this thread gets, the factor and the limit.
    uint32_t qb[kTiles][8][2];
    float qs[kTiles][2];
    int lim[kTiles][2];
    int min_lim = 0x7fffffff;
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      float top = 0.f;
      uint4 w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = lds128(smem_u32(query_base + ((turn & 1) * kMine + g + 8 * n) * kQueryLd + (4 * c + e) * 16));
      const uint32_t* ww = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 f = Pair<T>::get(ww[i]);
        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the row's largest value to [2^13, 2^14): what is not under 2^-27 of it keeps its bits
      const int shift = max(min(13 - ((__float_as_int(top) >> 23) - 127), 120), -115);
      const float f = __int_as_float((shift + 127) << 23);
#pragma unroll
      for (int i = 0; i < 16; ++i) {  // word i: dimensions 32c + 2i, 2i + 1; step i / 2
        const float2 v = Pair<T>::get(ww[i]);
        qb[n][i >> 1][i & 1] = half2_bits(v.x * f, v.y * f);
      }
      const float back = p.scale_log2 * __int_as_float((127 - shift) << 23);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        qs[n][y] = __shfl_sync(0xffffffffu, back, (2 * c + y) * 4);
        const int tok = (cur.rt * kMine + 8 * n + 2 * c + y) / p.group;
        lim[n][y] = 0;
        if (tok < s.count) {
          lim[n][y] = row_limit(s, tok);
          min_lim = min(min_lim, lim[n][y]);
        }
      }
    }
    min_lim = __reduce_min_sync(0xffffffffu, min_lim);
    if (lane == 0) mbar_arrive(&bar->q_empty[turn & 1]);

    float acc[kTiles][8][4];
    float m[kTiles][2], M[kTiles][2], l[kTiles][2];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][j][e] = 0.f;
#pragma unroll
      for (int y = 0; y < 2; ++y) m[n][y] = M[n][y] = kLowest, l[n][y] = 0.f;
    }

    for (int t = cur.t0; t < t1; ++t, ++it) {
      const int st = it % kStages;
      if (ok) ok = warp_wait(&bar->full[st], (it / kStages) & 1, p.status, kCacheTimeout);
      if (!ok) continue;
      const int key0 = t * kKeys + warp * kCacheBlock;
      if (key0 < s.len) {
        const uint32_t sk = smem_u32(smem + st * kStageBytes);
        // scores of keys g and g + 8: two chains of sums, since a product waits for the one before it
        float sacc[kTiles][2][4];
        {
          uint32_t kw[2][8];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int row = warp * kCacheBlock + 8 * y + g;
            const uint4 k0 = lds128(sk + row * 128 + (((2 * c) ^ (row & 7)) << 4));
            const uint4 k1 = lds128(sk + row * 128 + (((2 * c + 1) ^ (row & 7)) << 4));
            kw[y][0] = k0.x, kw[y][1] = k0.y, kw[y][2] = k0.z, kw[y][3] = k0.w;
            kw[y][4] = k1.x, kw[y][5] = k1.y, kw[y][6] = k1.z, kw[y][7] = k1.w;
          }
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sacc[n][0][e] = sacc[n][1][e] = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t a0 = f16_of_lo(kw[0][i]), a1 = f16_of_lo(kw[1][i]), a2 = f16_of_hi(kw[0][i]), a3 = f16_of_hi(kw[1][i]);
#pragma unroll
            for (int n = 0; n < kTiles; ++n) mma_f16(sacc[n][i & 1], a0, a1, a2, a3, qb[n][i][0], qb[n][i][1]);
          }
        }
        const float ks = block_scales[st * 8 + warp * 2], vs = block_scales[st * 8 + warp * 2 + 1];
        // log2 of the values' scale; NaN stays NaN
        const float ev = vs == vs ? (float)((__float_as_int(vs) >> 23) - 127) : vs;
        const bool edge = key0 + kCacheBlock > min_lim;
        float x[kTiles][4];  // keys g, g + 8 (e / 2), rows 2c, 2c + 1 (e % 2)
        bool grown = false;
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[n][e] = (sacc[n][0][e] + sacc[n][1][e]) * (qs[n][e & 1] * ks);
            if (edge && key0 + g + (e >> 1) * 8 >= lim[n][e & 1]) x[n][e] = -INFINITY;
            grown = grown || x[n][e] > m[n][e & 1] + kGrowth || x[n][e] + ev > M[n][e & 1] + kGrowth;
          }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float mx = fmaxf(x[n][y], x[n][2 + y]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              const float mn = fmaxf(m[n][y], mx), Mn = fmaxf(M[n][y], mx + ev);
              l[n][y] *= fast_exp2(m[n][y] - mn);
              const float f = fast_exp2(M[n][y] - Mn);
              m[n][y] = mn, M[n][y] = Mn;
#pragma unroll
              for (int j = 0; j < 8; ++j) acc[n][j][y] *= f, acc[n][j][2 + y] *= f;
            }
        }
        uint32_t pb[kTiles][2];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          float pv[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            l[n][e & 1] += fast_exp2(x[n][e] - m[n][e & 1]);
            pv[e] = fast_exp2(x[n][e] + (ev - M[n][e & 1]));
            if (edge && x[n][e] == -INFINITY) pv[e] = 0.f;  // also beside a poisoned block's NaN
          }
          pb[n][0] = transpose_8x8(half2_bits(pv[0], pv[1]));
          pb[n][1] = transpose_8x8(half2_bits(pv[2], pv[3]));
        }
        const uint32_t sv = sk + kHalfStage;
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = warp * kCacheBlock + 2 * c + (i & 1) + (i >> 1) * 8;
          v[i] = lds128(sv + row * 128 + ((g ^ (row & 7)) << 4));
          if (t * kKeys + row >= s.len) v[i] = make_uint4(0, 0, 0, 0);  // not written: any byte, NaN among them
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t w0 = (&v[0].x)[q], w1 = (&v[1].x)[q], w2 = (&v[2].x)[q], w3 = (&v[3].x)[q];
          const uint32_t lo01 = __byte_perm(w0, w1, 0x5140), lo23 = __byte_perm(w2, w3, 0x5140);
          const uint32_t hi01 = __byte_perm(w0, w1, 0x7362), hi23 = __byte_perm(w2, w3, 0x7362);
          const uint32_t a0 = f16_of_lo(lo01), a1 = f16_of_hi(lo01), a2 = f16_of_lo(lo23), a3 = f16_of_hi(lo23);
          const uint32_t b0 = f16_of_lo(hi01), b1 = f16_of_hi(hi01), b2 = f16_of_lo(hi23), b3 = f16_of_hi(hi23);
#pragma unroll
          for (int n = 0; n < kTiles; ++n) {
            mma_f16(acc[n][2 * q], a0, a1, a2, a3, pb[n][0], pb[n][1]);
            mma_f16(acc[n][2 * q + 1], b0, b1, b2, b3, pb[n][0], pb[n][1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->empty[st]);
    }

    // ---- join the four warps
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float sum = l[n][y];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int r = 8 * n + 2 * c + y;
        float* o = joined + (warp * kMine + r) * kOutLd + 16 * g;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<float4*>(o + 4 * q) = make_float4(acc[n][2 * q][y], acc[n][2 * q][2 + y], acc[n][2 * q + 1][y], acc[n][2 * q + 1][2 + y]);
        if (g == 0) {
          float* sp = stats + (warp * kMine + r) * 4;
          sp[0] = m[n][y], sp[1] = M[n][y], sp[2] = sum;
        }
      }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    constexpr int kPer = kMine * kCacheDim / (kWarps * 32);  // values of a thread: 8 or 16, of one row
    const int r = threadIdx.x * kPer / kCacheDim, d0 = threadIdx.x * kPer % kCacheDim;
    if (r < rows) {
      float mc = kLowest, sum = 0.f, f[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mc = fmaxf(mc, stats[(w * kMine + r) * 4]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* sp = stats + (w * kMine + r) * 4;
        sum += sp[2] * fast_exp2(sp[0] - mc);
        f[w] = sp[1] <= kLowest ? 0.f : exp2f(sp[1] - mc);  // back to the sum's maximum
      }
      float o[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) o[e] = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
#pragma unroll
        for (int e = 0; e < kPer; e += 4) {
          const float4 x = *reinterpret_cast<const float4*>(joined + (w * kMine + r) * kOutLd + d0 + e);
          o[e] += x.x * f[w], o[e + 1] += x.y * f[w], o[e + 2] += x.z * f[w], o[e + 3] += x.w * f[w];
        }
      if (cur.t0 == 0 && cur.t1 == cur.tiles) {
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        const int row = cur.rt * kMine + r;
        uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) +
                                              ((int64_t)(s.row + row / p.group) * p.H + cur.h * p.group + row % p.group) * kCacheDim + d0);
#pragma unroll
        for (int e = 0; e < kPer; e += 8)
          dst[e / 8] = make_uint4(Pair<T>::put(o[e] * inv, o[e + 1] * inv), Pair<T>::put(o[e + 2] * inv, o[e + 3] * inv),
                                  Pair<T>::put(o[e + 4] * inv, o[e + 5] * inv), Pair<T>::put(o[e + 6] * inv, o[e + 7] * inv));
      } else {
        const int64_t part = (int64_t)blockIdx.x * 2 + (cur.t0 == 0 ? 1 : 0);
        float4* dst = reinterpret_cast<float4*>(p.parts + (part * kRows + r) * kCacheDim + d0);
#pragma unroll
        for (int e = 0; e < kPer; e += 4) dst[e / 4] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        if (d0 == 0) p.part_ml[part * kRows + r] = make_float2(mc, sum);
      }
    }
    if (cur.t0 > 0 || cur.t1 < cur.tiles) {  // at most twice: the share's first segment and its last
      split[cur.t0 == 0 ? 1 : 0] = cur;
      has_split |= cur.t0 == 0 ? 2 : 1;
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");  // the buffer is free again
  }
  if (!has_split) return;
  // ---- The blocks of a segment lie side by side, from the one with its first tile to the one with its
  // last.  Parts are announced once, at the end of the share; who comes last joins them.
  __threadfence();
  asm volatile("bar.sync 1, 128;" ::: "memory");
  if (threadIdx.x < 2 && (has_split >> threadIdx.x & 1)) {
    const Segment& x = split[threadIdx.x];
    const int b0 = block_of(x.first_tile), b1 = block_of(x.first_tile + x.tiles - 1);
    const int before = atomicAdd(p.arrived + b0, 1);
    last_of[threadIdx.x] = before == b1 - b0 ? b0 : -1;
    if (before == b1 - b0) p.arrived[b0] = 0;
  }
  asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    if (!(has_split >> x & 1) || last_of[x] < 0) continue;
    __threadfence();
    const Seq s = walk.seq(split[x].i);
    const int rows = min(s.count * p.group - split[x].rt * kMine, kMine);
    join_parts<T, kMine>(p, split[x], s, rows, last_of[x], block_of(split[x].first_tile + split[x].tiles - 1), warp, lane);
  }
}

template <int kTiles>
constexpr size_t smem_bytes() {
  using S = Shape<kTiles>;
  return 1024 + S::kStages * kStageBytes + sizeof(float) * (kWarps * S::kRowsHeld * (kOutLd + 4) + S::kStages * 8) +
         2 * S::kRowsHeld * kQueryLd + sizeof(Barriers<S::kStages>) + sizeof(Seq) * kWindow;
}

template <typename T, int kTiles>
cudaError_t launch(const CUtensorMap& map, const Params& p, int grid, cudaStream_t stream) {
  static bool set[64] = {false};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (!set[dev]) {
    err = cudaFuncSetAttribute(cache_attention_kernel<T, kTiles>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)smem_bytes<kTiles>());
    if (err != cudaSuccess) return err;
    set[dev] = true;
  }
  grid = std::min(grid, Shape<kTiles>::kBlocksPerSm * 148);
  return launch_after_previous(cache_attention_kernel<T, kTiles>, grid, kThreads, smem_bytes<kTiles>(), stream, map, p);
}

}  // namespace

namespace mimir {
cudaError_t launch_cache_attention(const CUtensorMap& map, const AttentionParams& p, bool bf16, bool full, int grid,
                                   cudaStream_t stream) {
  if (bf16) return full ? launch<__nv_bfloat16, 2>(map, p, grid, stream) : launch<__nv_bfloat16, 1>(map, p, grid, stream);
  return full ? launch<__half, 2>(map, p, grid, stream) : launch<__half, 1>(map, p, grid, stream);
}
}  // namespace mimir
