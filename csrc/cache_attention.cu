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
// sums, which a second kernel joins in the order of the keys (no atomics: results do not depend on
// scheduling).
//
// Matrix products are m16n8k16 with fp16 operands and fp32 sums.  Bytes become fp16 exactly; the
// scales, powers of two, stay outside: a key block's multiplies its scores, a value block's enters
// the exponent of the probability that multiplies the values, exp2(x + ev - M) with a maximum M of
// x + ev of its own (so it neither overflows nor loses small weights), beside exp2(x - m) for the
// sum.  Probabilities are rounded to fp16 (11 bits) for the product.  Query rows are shifted by a
// power of two into fp16's range, so that bf16 rows keep all their bits.
// The contraction over the head dimension may run in any order: thread c of a quad takes the bytes
// 32c..32c+31 of a key row, which two 16-byte loads bring without bank conflicts under the swizzle, and
// the same dimensions of the query rows.  Of the values it takes 16 bytes of four rows; output column
// 16 g + j belongs to column g of product j.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "kv_cache.cuh"
#include "tma.cuh"

using namespace mimir;

namespace {

constexpr int kKeys = 64;                      // keys of a unit
constexpr int kStages = 4;
constexpr int kWarps = 4;                      // consumers
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kRows = 16;                      // rows of a tile
constexpr uint32_t kHalfStage = kKeys * kCacheDim;
constexpr uint32_t kStageBytes = 2 * kHalfStage;
constexpr int kMaxSeqs = 1024;                 // sequences of one launch
constexpr int kOutLd = 132;                    // floats of a row in the join buffer
constexpr float kLowest = -3e38f;
constexpr float kGrowth = 8.f;                 // maxima move only when they grow by more than 2^8

struct Params {
  const void* q;
  int64_t q_tok, q_head;
  void* out;                                   // [tokens, H, 128]
  const float* scales;
  const int *table, *lens, *seqs, *cu, *prefix;
  int slots, width, n, tokens, H, KV, group, page, page_shift, npages;
  float scale_log2;
  int4* desc;                                  // per block: the segment that it begins and others finish
  float* parts;                                // [blocks][2][16][128]
  float2* part_ml;                             // [blocks][2][16]: maximum and sum
  int last_batch;
  int* status;
};

struct __align__(8) Barriers {
  uint64_t full[kStages];
  uint64_t empty[kStages];
};

struct Seq {
  int len, row, count, slot;  // tokens, first new row, new rows, page table row
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
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
__device__ __forceinline__ int row_limit(const Seq& s, int prefix, int tok) {
  const int pos = s.len - s.count + tok;
  int lim = pos + 1;
  if (pos < prefix) lim = max(lim, prefix);
  return max(min(lim, s.len), 0);
}

// A share of the line of units, one segment at a time.
struct Walk {
  const int64_t* first;  // units before a sequence
  const Seq* seqs;
  int n, KV, group;
  int64_t u, end;
  int i;
  // the segment
  int h, rt, t0, t1, tiles;
  int64_t seg_begin;
  __device__ void start() {
    int lo = 0, hi = n - 1;  // the last sequence with first <= u (empty ones have no units)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= u) lo = mid;
      else hi = mid - 1;
    }
    i = lo;
  }
  __device__ bool next() {
    if (u >= end) return false;
    while (first[i + 1] <= u) ++i;
    const Seq& s = seqs[i];
    const int rts = (s.count * group + kRows - 1) / kRows;
    tiles = max((s.len + kKeys - 1) / kKeys, 1);
    const int64_t local = u - first[i];
    const int64_t seg = local / tiles;
    t0 = (int)(local % tiles);
    h = (int)(seg / rts);
    rt = (int)(seg % rts);
    seg_begin = u - t0;
    t1 = (int)min((int64_t)tiles, t0 + (end - u));
    u += t1 - t0;
    return true;
  }
};

template <typename T, bool kFull>
__global__ void __launch_bounds__(kThreads) cache_attention_kernel(const __grid_constant__ CUtensorMap map, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int kMine = kFull ? 16 : 8;  // rows of a tile that can hold queries
  float* joined = reinterpret_cast<float*>(smem + kStages * kStageBytes);        // [kWarps][kMine][kOutLd]
  float* stats = joined + kWarps * kMine * kOutLd;                               // [kWarps][kMine][4]: m, M, l
  float* block_scales = stats + kWarps * kMine * 4;                              // [kStages][4 blocks][k, v]
  Barriers* bar = reinterpret_cast<Barriers*>(block_scales + kStages * 8);
  int64_t* first = reinterpret_cast<int64_t*>(bar + 1);                          // [n + 1]
  Seq* seqs = reinterpret_cast<Seq*>(first + p.n + 1);                           // [n]
  __shared__ int64_t scan_sums[kThreads / 32];
  __shared__ int64_t scan_base;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bar->full[s], 1 + 8);
      mbar_init(&bar->empty[s], kWarps);
    }
    fence_mbarrier_init();
    tma_prefetch_desc(&map);
    scan_base = 0;
  }
  // ---- the line of units
  for (int base = 0; base < p.n; base += kThreads) {
    const int i = base + (int)threadIdx.x;
    int64_t units = 0;
    if (i < p.n) {
      Seq s;
      s.row = p.cu[i];
      s.count = max(min(p.cu[i + 1], p.tokens) - s.row, 0);
      if (s.row < 0) s.count = 0;
      s.slot = p.seqs[i];
      s.len = 0;
      if (s.slot < 0 || s.slot >= p.slots) {
        s.slot = 0;
        if (s.count > 0) record_status(p.status, kCacheBadSlot);
      } else {
        s.len = p.lens[s.slot];
        if (s.len < s.count) record_status(p.status, kCacheBadLength);
        if (s.len < 0) s.len = 0;
        if (s.len > p.width * p.page) {
          s.len = p.width * p.page;
          record_status(p.status, kCacheBadPage);
        }
      }
      seqs[i] = s;
      units = (int64_t)p.KV * ((s.count * p.group + kRows - 1) / kRows) * max((s.len + kKeys - 1) / kKeys, 1);
    }
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
  if (threadIdx.x == 0) {
    first[p.n] = scan_base;
    p.desc[blockIdx.x] = make_int4(-1, 0, 0, 0);
  }
  __syncthreads();
  const int64_t total = p.n > 0 ? first[p.n] : 0;
  // rows that belong to no sequence
  if (p.last_batch) {
    const int from = p.n > 0 ? min(max(p.cu[p.n], 0), p.tokens) : 0;
    uint4* o = reinterpret_cast<uint4*>(p.out);
    const int64_t per = (int64_t)p.H * kCacheDim * sizeof(T) / 16;
    for (int64_t k = from * per + blockIdx.x * (int64_t)kThreads + threadIdx.x; k < p.tokens * per; k += (int64_t)gridDim.x * kThreads)
      o[k] = make_uint4(0, 0, 0, 0);
  }
  const int64_t blocks = min((int64_t)gridDim.x, total);
  if (blockIdx.x >= blocks) return;
  Walk walk{first, seqs, p.n, p.KV, p.group};
  const int64_t u0 = total * blockIdx.x / blocks;
  walk.u = u0;
  walk.end = total * (blockIdx.x + 1) / blocks;
  walk.start();
  const int piece = min(p.page, kKeys), pieces = kKeys / piece;  // keys that lie together, and their number in a unit

  // The tiles that a row tile needs: keys up to the largest limit of its rows.
  auto tiles_needed = [&](const Seq& s, int prefix, int rt) {
    const int last = min((rt * kRows + kRows - 1) / p.group, s.count - 1);
    int lim = row_limit(s, prefix, last);
    if (prefix > 0) lim = max(lim, row_limit(s, prefix, rt * kRows / p.group));
    return (lim + kKeys - 1) / kKeys;
  };

  if (warp == kWarps) {
    // ------------------------------------------------------------ producer
    int it = 0;
    bool ok = true;
    while (ok && walk.next()) {
      const Seq s = seqs[walk.i];
      const int prefix = p.prefix != nullptr ? p.prefix[walk.i] : 0;
      const int t1 = min(walk.t1, tiles_needed(s, prefix, walk.rt));
      const int* row = p.table + (int64_t)s.slot * p.width;
      int base = -32, mine = -1;  // page ids of the pieces base .. base + 31, one a lane
      for (int t = walk.t0; ok && t < t1; ++t, ++it) {
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
        const float* src = p.scales + (((int64_t)page_b * 2 + (lane & 1)) * p.KV + walk.h) * (p.page / kCacheBlock) +
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
            tma_load_3d(dst, &map, &bar->full[st], 0, (t * kKeys + x * piece) & (p.page - 1), (page * 2 + lane) * p.KV + walk.h);
          }
          __syncwarp();
        }
      }
    }
    // no copy into this block's shared memory may outlive it
    asm volatile("cp.async.wait_all;" ::: "memory");
    for (int j = max(0, it - kStages); j < it; ++j) warp_wait(&bar->full[j % kStages], (j / kStages) & 1, p.status, kCacheTimeout);
    return;
  }

  // -------------------------------------------------------------- consumers
  const int g = lane >> 2, c = lane & 3;
  int it = 0;
  bool ok = true;
  while (walk.next()) {
    const Seq s = seqs[walk.i];
    const int prefix = p.prefix != nullptr ? p.prefix[walk.i] : 0;
    const int t1 = min(walk.t1, tiles_needed(s, prefix, walk.rt));
    const int rows = min(s.count * p.group - walk.rt * kRows, kRows);
    // query rows g and g + 8 of the tile: dimensions 32c .. 32c + 31
    uint32_t qa[8][kFull ? 4 : 2];
    float qs[kFull ? 2 : 1];
    int lim[kFull ? 2 : 1];
    int min_lim = 0x7fffffff;
#pragma unroll
    for (int x = 0; x < (kFull ? 2 : 1); ++x) {
      const int r = walk.rt * kRows + g + 8 * x;
      const int tok = r / p.group, head = walk.h * p.group + r % p.group;
      uint4 w[4] = {};
      lim[x] = 0;
      if (tok < s.count) {
        const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + (int64_t)(s.row + tok) * p.q_tok +
                                                          head * p.q_head + 32 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = src[i];
        lim[x] = row_limit(s, prefix, tok);
        min_lim = min(min_lim, lim[x]);
      }
      float top = 0.f;
      const uint32_t* ww = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 f = Pair<T>::get(ww[i]);
        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the row's largest value to [2^13, 2^14): a power of two, nothing is rounded away
      const int shift = max(min(13 - ((__float_as_int(top) >> 23) - 127), 120), -115);
      const float f = __int_as_float((shift + 127) << 23);
      qs[x] = p.scale_log2 * __int_as_float((127 - shift) << 23);
#pragma unroll
      for (int i = 0; i < 16; ++i) {  // word i: dimensions 32c + 2i, 2i + 1; step i / 2
        const float2 v = Pair<T>::get(ww[i]);
        qa[i >> 1][(i & 1) * (kFull ? 2 : 1) + x] = half2_bits(v.x * f, v.y * f);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) min_lim = min(min_lim, __shfl_xor_sync(0xffffffffu, min_lim, o));

    float acc[16][4];
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
    constexpr int R = kFull ? 2 : 1;
    float m[R], M[R], l[R];
#pragma unroll
    for (int x = 0; x < R; ++x) m[x] = M[x] = kLowest, l[x] = 0.f;

    for (int t = walk.t0; t < t1; ++t, ++it) {
      const int st = it % kStages;
      if (ok) ok = warp_wait(&bar->full[st], (it / kStages) & 1, p.status, kCacheTimeout);
      if (!ok) continue;
      const int key0 = t * kKeys + warp * kCacheBlock;
      if (key0 < s.len) {
        const uint32_t sk = smem_u32(smem + st * kStageBytes);
        float sacc[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) sacc[nt][e] = 0.f;
          const int row = warp * kCacheBlock + nt * 8 + g;
          const uint4 k0 = lds128(sk + row * 128 + (((2 * c) ^ (row & 7)) << 4));
          const uint4 k1 = lds128(sk + row * 128 + (((2 * c + 1) ^ (row & 7)) << 4));
          const uint32_t kw[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
#pragma unroll
          for (int i = 0; i < 8; ++i)
            mma_f16(sacc[nt], qa[i][0], kFull ? qa[i][1] : 0u, qa[i][kFull ? 2 : 1], kFull ? qa[i][3] : 0u, f16_of_lo(kw[i]),
                    f16_of_hi(kw[i]));
        }
        const float ks = block_scales[st * 8 + warp * 2], vs = block_scales[st * 8 + warp * 2 + 1];
        // log2 of the values' scale; NaN stays NaN
        const float ev = vs == vs ? (float)((__float_as_int(vs) >> 23) - 127) : vs;
        const bool edge = key0 + kCacheBlock > min_lim;
        float pw[R][4], pv[R][4];
#pragma unroll
        for (int x = 0; x < R; ++x) {
          const float f = qs[x] * ks;
          float xs[4] = {sacc[0][2 * x] * f, sacc[0][2 * x + 1] * f, sacc[1][2 * x] * f, sacc[1][2 * x + 1] * f};
          if (edge) {
            const int rel = lim[x] - key0 - 2 * c;
            xs[0] = rel > 0 ? xs[0] : -INFINITY;
            xs[1] = rel > 1 ? xs[1] : -INFINITY;
            xs[2] = rel > 8 ? xs[2] : -INFINITY;
            xs[3] = rel > 9 ? xs[3] : -INFINITY;
          }
          float mx = fmaxf(fmaxf(xs[0], xs[1]), fmaxf(xs[2], xs[3]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float my = mx + ev;
          if (__any_sync(0xffffffffu, mx > m[x] + kGrowth || my > M[x] + kGrowth)) {
            const float mn = fmaxf(m[x], mx), Mn = fmaxf(M[x], my);
            l[x] *= fast_exp2(m[x] - mn);
            const float a = fast_exp2(M[x] - Mn);
            m[x] = mn, M[x] = Mn;
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[j][2 * x] *= a, acc[j][2 * x + 1] *= a;
          }
          const float shift = ev - M[x];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            pw[x][e] = fast_exp2(xs[e] - m[x]);
            pv[x][e] = fast_exp2(xs[e] + shift);
            if (edge && xs[e] == -INFINITY) pv[x][e] = 0.f;  // also beside a poisoned block's NaN
            l[x] += pw[x][e];
          }
        }
        const uint32_t a0 = half2_bits(pv[0][0], pv[0][1]), a2 = half2_bits(pv[0][2], pv[0][3]);
        const uint32_t a1 = kFull ? half2_bits(pv[R - 1][0], pv[R - 1][1]) : 0u, a3 = kFull ? half2_bits(pv[R - 1][2], pv[R - 1][3]) : 0u;
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
          mma_f16(acc[4 * q], a0, a1, a2, a3, f16_of_lo(lo01), f16_of_lo(lo23));
          mma_f16(acc[4 * q + 1], a0, a1, a2, a3, f16_of_hi(lo01), f16_of_hi(lo23));
          mma_f16(acc[4 * q + 2], a0, a1, a2, a3, f16_of_lo(hi01), f16_of_lo(hi23));
          mma_f16(acc[4 * q + 3], a0, a1, a2, a3, f16_of_hi(hi01), f16_of_hi(hi23));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->empty[st]);
    }

    // ---- join the four warps
#pragma unroll
    for (int x = 0; x < R; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      const int r = g + 8 * x;
      float* o = joined + (warp * kMine + r) * kOutLd + 32 * c;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int q = (k + c) & 3;  // spreads the quad over the banks
#pragma unroll
        for (int qq = 0; qq < 4; ++qq) {
          if (qq != q) continue;
          *reinterpret_cast<float4*>(o + 4 * qq) = make_float4(acc[4 * qq][2 * x], acc[4 * qq + 1][2 * x], acc[4 * qq + 2][2 * x], acc[4 * qq + 3][2 * x]);
          *reinterpret_cast<float4*>(o + 16 + 4 * qq) = make_float4(acc[4 * qq][2 * x + 1], acc[4 * qq + 1][2 * x + 1], acc[4 * qq + 2][2 * x + 1], acc[4 * qq + 3][2 * x + 1]);
        }
      }
      if (c == 0) {
        float* sp = stats + (warp * kMine + r) * 4;
        sp[0] = m[x], sp[1] = M[x], sp[2] = l[x];
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
      const bool begins = walk.t0 == 0, ends = walk.t1 == walk.tiles;
      if (begins && ends) {
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        const int row = walk.rt * kRows + r;
        uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) +
                                              ((int64_t)(s.row + row / p.group) * p.H + walk.h * p.group + row % p.group) * kCacheDim + d0);
#pragma unroll
        for (int e = 0; e < kPer; e += 8)
          dst[e / 8] = make_uint4(Pair<T>::put(o[e] * inv, o[e + 1] * inv), Pair<T>::put(o[e + 2] * inv, o[e + 3] * inv),
                                  Pair<T>::put(o[e + 4] * inv, o[e + 5] * inv), Pair<T>::put(o[e + 6] * inv, o[e + 7] * inv));
      } else {
        const int64_t part = (int64_t)blockIdx.x * 2 + (begins ? 1 : 0);
        float4* dst = reinterpret_cast<float4*>(p.parts + (part * kRows + r) * kCacheDim + d0);
#pragma unroll
        for (int e = 0; e < kPer; e += 4) dst[e / 4] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        if (d0 == 0) p.part_ml[part * kRows + r] = make_float2(mc, sum);
        if (threadIdx.x == 0 && begins) {
          // the block that holds the segment's last unit
          const int64_t last = walk.seg_begin + walk.tiles - 1;
          p.desc[blockIdx.x] = make_int4(walk.i, walk.h, walk.rt, (int)(((last + 1) * blocks - 1) / total));
        }
      }
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");  // the buffer is free again
  }
}

// Joins the partial sums of the segment that block `blockIdx.x` of the first kernel began.
template <typename T>
__global__ void __launch_bounds__(512) cache_attention_join_kernel(const Params p) {
  const int4 d = p.desc[blockIdx.x];
  if (d.x < 0) return;
  const int first_row = p.cu[d.x], count = min(p.cu[d.x + 1], p.tokens) - first_row;
  const int rows = min(count * p.group - d.z * kRows, kRows);
  const int col = threadIdx.x & 127;
  for (int r = threadIdx.x >> 7; r < rows; r += 4) {
    float m = kLowest, sum = 0.f, o = 0.f;
    for (int b = blockIdx.x; b <= d.w; ++b) {
      const int64_t part = (int64_t)b * 2 + (b == (int)blockIdx.x ? 1 : 0);
      const float2 ml = p.part_ml[part * kRows + r];
      const float x = p.parts[(part * kRows + r) * kCacheDim + col];
      const float mn = fmaxf(m, ml.x);
      const float fa = fast_exp2(m - mn), fb = fast_exp2(ml.x - mn);
      sum = sum * fa + ml.y * fb;
      o = o * fa + x * fb;
      m = mn;
    }
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    const int row = d.z * kRows + r;
    T* dst = reinterpret_cast<T*>(p.out) + ((int64_t)(first_row + row / p.group) * p.H + d.y * p.group + row % p.group) * kCacheDim;
    dst[col] = Pair<T>::one(o * inv);
  }
}

CUtensorMap pages_map(const at::Tensor& pages) {
  const int64_t rows = pages.size(3), heads = pages.size(0) * 2 * pages.size(2);
  bind_device_context();
  CUtensorMap map;
  cuuint64_t dims[3] = {(cuuint64_t)kCacheDim, (cuuint64_t)rows, (cuuint64_t)heads};
  cuuint64_t strides[2] = {(cuuint64_t)kCacheDim, (cuuint64_t)(rows * kCacheDim)};
  cuuint32_t box[3] = {(cuuint32_t)kCacheDim, (cuuint32_t)std::min<int64_t>(rows, kKeys), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = tensor_map_encoder()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, pages.data_ptr(), dims, strides, box, estr,
                                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled (pages) failed with code ", (int)r);
  return map;
}

size_t smem_bytes(bool full, int n) {
  const int mine = full ? 16 : 8;
  return 1024 + kStages * kStageBytes + sizeof(float) * (kWarps * mine * (kOutLd + 4) + kStages * 8) + sizeof(Barriers) +
         sizeof(int64_t) * (n + 1) + sizeof(Seq) * n;
}

template <typename T, bool kFull>
void launch(const CUtensorMap& map, const Params& p, int grid) {
  static bool set[64] = {false};
  int dev = 0;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  if (!set[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(cache_attention_kernel<T, kFull>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)smem_bytes(kFull, kMaxSeqs)));
    set[dev] = true;
  }
  auto st = at::cuda::getCurrentCUDAStream();
  cache_attention_kernel<T, kFull><<<grid, kThreads, smem_bytes(kFull, p.n), st>>>(map, p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  cache_attention_join_kernel<T><<<grid, 512, 0, st>>>(p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace

at::Tensor cache_attention(at::Tensor q, at::Tensor pages, at::Tensor scales, at::Tensor table, at::Tensor lens,
                           at::Tensor seqs, at::Tensor cu_new, c10::optional<at::Tensor> prefix_lens,
                           double softmax_scale, int64_t max_new) {
  check_pool(pages, scales, 0);
  const at::Device dev = pages.device();
  check_rows(q, "q", dev);
  check_batch(table, lens, seqs, cu_new, dev);
  const int64_t H = q.size(1), KV = pages.size(2);
  CACHE_CHECK(H >= 1 && H % KV == 0, "query heads ", H, " must be divisible by key/value heads ", KV);
  CACHE_CHECK(q.size(0) * (H / KV) < (int64_t(1) << 31) - 64, "too many query rows");
  CACHE_CHECK(table.size(1) * pages.size(3) < (int64_t(1) << 31) - 4096, "sequences of 2^31 tokens or more");
  if (prefix_lens.has_value()) {
    check_int32(*prefix_lens, "prefix_lens", 1, dev);
    CACHE_CHECK(prefix_lens->size(0) == seqs.size(0), "prefix_lens needs one length for each of seqs");
  }
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor out = at::empty({q.size(0), H, kCacheDim}, q.options());
  const int64_t n = seqs.size(0);
  if (q.size(0) == 0) return out;
  if (n == 0 || pages.size(0) == 0) return out.zero_();
  const CUtensorMap map = pages_map(pages);
  Params p{};
  p.q = q.data_ptr();
  p.q_tok = q.stride(0), p.q_head = q.stride(1);
  p.out = out.data_ptr();
  p.scales = scales.data_ptr<float>();
  p.table = table.data_ptr<int>(), p.lens = lens.data_ptr<int>();
  p.slots = (int)table.size(0), p.width = (int)table.size(1), p.tokens = (int)q.size(0);
  p.H = (int)H, p.KV = (int)KV, p.group = (int)(H / KV);
  p.page = (int)pages.size(3), p.page_shift = __builtin_ctz(p.page), p.npages = (int)pages.size(0);
  p.scale_log2 = (float)(softmax_scale * 1.4426950408889634);
  p.status = cache_status_word(dev);
  const bool full = max_new < 1 || max_new * p.group > 8;
  for (int64_t base = 0; base < n; base += kMaxSeqs) {
    p.n = (int)std::min<int64_t>(kMaxSeqs, n - base);
    p.seqs = seqs.data_ptr<int>() + base;
    p.cu = cu_new.data_ptr<int>() + base;
    p.prefix = prefix_lens.has_value() ? prefix_lens->data_ptr<int>() + base : nullptr;
    p.last_batch = base + p.n == n;
    // no more blocks than units: at most this many
    const int64_t row_tiles = std::min<int64_t>(q.size(0), p.n) + q.size(0) * p.group / kRows + 1;
    const int64_t most = row_tiles * KV * ((p.width * p.page + kKeys - 1) / kKeys + 1);
    const int grid = (int)std::min<int64_t>(2 * 148, std::max<int64_t>(most, 1));
    at::Tensor work = at::empty({grid * (int64_t)(4 + 2 * kRows * (kCacheDim + 2))}, q.options().dtype(at::kFloat));
    float* w = work.data_ptr<float>();
    p.desc = reinterpret_cast<int4*>(w);
    p.parts = w + grid * 4;
    p.part_ml = reinterpret_cast<float2*>(p.parts + (int64_t)grid * 2 * kRows * kCacheDim);
    if (q.scalar_type() == at::kBFloat16)
      full ? launch<__nv_bfloat16, true>(map, p, grid) : launch<__nv_bfloat16, false>(map, p, grid);
    else
      full ? launch<__half, true>(map, p, grid) : launch<__half, false>(map, p, grid);
  }
  return out;
}
