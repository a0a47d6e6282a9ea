// The 8-bit paged key/value cache: rotary + quantise + write (cache_append), and the bookkeeping
// and movement of its pages (cache_reserve, cache_free, cache_fork, cache_compact, cache_copy).
// Layout and status codes: serving.h.
//
// Append.  A new token at position p gets x' = x * cos[p] + rot(x) * sin[p] (k and q; the two
// products and their sum each rounded to fp32) and v' = v.  All new tokens of one head in one
// block of 16 share the scale 2^e with e the smallest exponent (>= -32) such that no |x'| is over
// 448 * 2^e, and not below the exponent of the tokens that the block already holds; where those
// held a smaller one, their bytes are rounded again to the new one.  Powers of two make every
// product and quotient with a scale exact, so a value is rounded once (e4m3, nearest even), and
// a token whose block later grows is rounded again only where it falls below the normal range.
// Measured on B200: 13703 tokens of five prompts, 16 and 4 heads: 40 us for 168 MB (4.1 TB/s; with four heads
// a block and three blocks an SM 56 us: time goes on waiting for loads, so threads count); 64 sequences' next
// tokens: 5 us.
//
// Pages.  One block keeps the books (sums over the batch, free pages lowest first by a scan of the counts), so
// that results do not depend on scheduling; a second launch moves the bytes.  4 prompts forked to 32 slots over 24
// layers: 17 us, of it some 5 for the books, for 50 MB written; 195 pages of 24 layers into another pool: 110 us
// (5.5 TB/s read and written).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "serving.h"

using namespace mimir;

namespace {

__device__ int g_cache_status;

__device__ __forceinline__ void report(int* status, int code) { atomicCAS(status, 0, code); }

template <typename T>
__device__ __forceinline__ uint2 raw4(const T* p) {
  return *reinterpret_cast<const uint2*>(p);
}
template <typename T>
__device__ __forceinline__ float4 widen(uint2 w);
template <>
__device__ __forceinline__ float4 widen<__nv_bfloat16>(uint2 w) {
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
template <>
__device__ __forceinline__ float4 widen<__half>(uint2 w) {
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
  uint2 w;
  *reinterpret_cast<__nv_bfloat162*>(&w.x) = __floats2bfloat162_rn(v.x, v.y);
  *reinterpret_cast<__nv_bfloat162*>(&w.y) = __floats2bfloat162_rn(v.z, v.w);
  *reinterpret_cast<uint2*>(p) = w;
}
__device__ __forceinline__ void store4(__half* p, float4 v) {
  uint2 w;
  *reinterpret_cast<__half2*>(&w.x) = __floats2half2_rn(v.x, v.y);
  *reinterpret_cast<__half2*>(&w.y) = __floats2half2_rn(v.z, v.w);
  *reinterpret_cast<uint2*>(p) = w;
}

__device__ __forceinline__ float turn(float x, float other, float c, float s) {
  return __fadd_rn(__fmul_rn(x, c), __fmul_rn(other, s));
}

// Rotates four dimensions d (lo) and their partners d + 64 (hi).
__device__ __forceinline__ void rotate(float4& lo, float4& hi, float4 cl, float4 ch, float4 sl, float4 sh) {
  const float4 l = lo, h = hi;
  lo = make_float4(turn(l.x, -h.x, cl.x, sl.x), turn(l.y, -h.y, cl.y, sl.y), turn(l.z, -h.z, cl.z, sl.z),
                   turn(l.w, -h.w, cl.w, sl.w));
  hi = make_float4(turn(h.x, l.x, ch.x, sh.x), turn(h.y, l.y, ch.y, sh.y), turn(h.z, l.z, ch.z, sh.z),
                   turn(h.w, l.w, ch.w, sh.w));
}

// Smallest e >= kCacheMinExp with amax <= 448 * 2^e (448 = 1.75 * 2^8), amax finite.
__device__ __forceinline__ int scale_exponent(float amax) {
  const int bits = __float_as_int(amax);
  const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000);
  return max(e, kCacheMinExp);
}
__device__ __forceinline__ float two_to(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// Four values as e4m3 bytes (nearest even).
__device__ __forceinline__ uint32_t to_e4m3(float4 v) {
  const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(v.x, v.y), __NV_SATFINITE, __NV_E4M3);
  const uint32_t b = __nv_cvt_float2_to_fp8x2(make_float2(v.z, v.w), __NV_SATFINITE, __NV_E4M3);
  return a | (b << 16);
}
__device__ __forceinline__ float4 from_e4m3(uint32_t w) {
  const __half2 a(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffff), __NV_E4M3));
  const __half2 b(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3));
  const float2 x = __half22float2(a), y = __half22float2(b);
  return make_float4(x.x, x.y, y.x, y.y);
}
__device__ __forceinline__ float4 times(float4 v, float f) { return make_float4(v.x * f, v.y * f, v.z * f, v.w * f); }

// The largest magnitude, as bits; a value that is not finite becomes zero and is reported in `bad`.
__device__ __forceinline__ uint32_t take_finite(float4& v, bool& bad) {
  float* x = reinterpret_cast<float*>(&v);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!(fabsf(x[i]) <= 3.402823466e38f)) {
      x[i] = 0.f;
      bad = true;
    }
    top = max(top, __float_as_uint(fabsf(x[i])));
  }
  return top;
}

constexpr int kAppendThreads = 256;
constexpr int kTeams = kAppendThreads / 16;  // a team of 16 lanes holds one row of a head
constexpr int kHeads = 2;                    // key/value heads of a thread block

// One block of 16 cached tokens (those of its tokens that are new) and up to two key/value heads with
// their query heads.  Thread block b finds its tokens itself: sequence i has at most
// new / 16 + 2 blocks, so the ones from cu[i] / 16 + 3 i on are its own, and a few stay empty.  After that
// all loads are under way at once.  A team has one row: sixteen rows give it all heads of its row, one
// row is shared by all teams, a head each.
template <typename T>
__global__ void __launch_bounds__(kAppendThreads, 4) cache_append_kernel(const AppendParams p) {
  __shared__ int at_row, at_pos, at_page, at_rows, at_written;  // first new row, its position, page, rows, rows written
  __shared__ uint32_t tops[kHeads][2];                          // largest magnitude, keys and values
  __shared__ int exponents[kHeads][2], poisoned[kHeads][2];
  const int lane = threadIdx.x & 31, team = threadIdx.x >> 4, d = (threadIdx.x & 15) * 4;
  after_previous();
  if (threadIdx.x < 32) {
    const int b = blockIdx.x;
    int lo = 0, size = p.n + 1;  // the last i with cu[i] / 16 + 3 i <= b, 32 candidates a step
    while (size > 1) {
      const int step = (size + 31) / 32;
      const int at = min(lo + lane * step, p.n);
      const int c = __popc(__ballot_sync(0xffffffffu, lo + lane * step < lo + size && max(p.cu[at], 0) / kCacheBlock + 3 * at <= b));
      const int next = lo + max(c - 1, 0) * step;
      size = min(step, lo + size - next);
      lo = next;
    }
    if (lane == 0) {
      int rows = 0, written = 0, row = 0, pos = 0, page = -1;
      if (lo < p.n) {
        const NewRows own = new_rows(p.cu, lo, p.tokens);
        const int first = own.first, count = own.count, slot = p.seqs[lo];
        const int j = b - (max(p.cu[lo], 0) / kCacheBlock + 3 * lo);
        const bool good = slot >= 0 && slot < p.slots;
        const int start = good ? p.lens[slot] - count : 0;
        if (own.good && good && start >= 0) {
          const int64_t block = (int64_t)(start / kCacheBlock + j) * kCacheBlock;
          const int64_t from = max(block, (int64_t)start), to = min(block + kCacheBlock, (int64_t)start + count);
          rows = (int)max(to - from, (int64_t)0);
          pos = (int)from;
          row = first + pos - start;
          written = (int)min(max(p.positions - from, (int64_t)0), (int64_t)rows);
          if (written < rows) report(p.status, kCacheBadLength);
          if (rows > 0) {
            const int x = pos / p.page;
            page = x < p.width ? p.table[(int64_t)slot * p.width + x] : -1;
            if (page < 0 || page >= p.npages) {
              report(p.status, kCacheBadPage);
              page = -1;
            }
          }
        } else if (j >= 0) {  // its rows become zeros
          rows = min(max(count - j * kCacheBlock, 0), kCacheBlock);
          row = first + j * kCacheBlock;
          if (rows > 0) report(p.status, good ? kCacheBadLength : kCacheBadSlot);
        }
      }
      at_rows = rows, at_written = written, at_row = row, at_pos = pos, at_page = page;
    }
  } else if (threadIdx.x < 32 + 2 * kHeads) {
    (&tops[0][0])[threadIdx.x - 32] = 0;
    (&poisoned[0][0])[threadIdx.x - 32] = 0;
  }
  if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0) {  // rows that belong to no sequence; all bounds
    uint4* o = reinterpret_cast<uint4*>(p.q_out);
    const int64_t per = (int64_t)p.H * kCacheDim / 8;
    const int64_t before = (p.n > 0 ? min(p.cu[0], p.tokens) : 0) * per;
    const int64_t from = (p.n > 0 ? min(max(p.cu[p.n], 0), p.tokens) : 0) * per;
    for (int64_t x = threadIdx.x; x < before; x += kAppendThreads) o[x] = make_uint4(0, 0, 0, 0);
    for (int64_t x = from + threadIdx.x; x < p.tokens * per; x += kAppendThreads) o[x] = make_uint4(0, 0, 0, 0);
    check_bounds(p.cu, p.n, p.tokens, p.status);
  }
  __syncthreads();
  const int rows = at_rows, written = at_written, pos0 = at_pos, page = at_page;
  if (rows == 0) return;
  const int h0 = blockIdx.y * kHeads, heads = min(kHeads, p.KV - h0), group = p.H / p.KV;
  const T* k = reinterpret_cast<const T*>(p.k) + at_row * p.k_tok + h0 * p.k_head + d;
  const T* v = reinterpret_cast<const T*>(p.v) + at_row * p.v_tok + h0 * p.v_head + d;
  const T* q = reinterpret_cast<const T*>(p.q) + at_row * p.q_tok + (int64_t)h0 * group * p.q_head + d;
  T* out = reinterpret_cast<T*>(p.q_out) + ((int64_t)at_row * p.H + (int64_t)h0 * group) * kCacheDim + d;
  const float* cos = p.cos + (int64_t)pos0 * kCacheDim + d;
  const float* sin = p.sin + (int64_t)pos0 * kCacheDim + d;
  const int writes = page >= 0 ? written : 0;

  // Team -> row r and the heads sub, sub + subs, ...: as many teams a row as a power of two allows.
  const int shift = rows > 8 ? 4 : rows > 4 ? 3 : rows > 2 ? 2 : rows > 1 ? 1 : 0;
  const int r = team & ((1 << shift) - 1), sub = team >> shift, subs = kTeams >> shift;
  const bool writing = r < writes, reading = r < written;
  const T* kr = k + r * p.k_tok;
  const T* vr = v + r * p.v_tok;
  const T* qr = q + r * p.q_tok;
  // ---- keys and values, held as they are until their scale is known
  uint2 kraw[kHeads][2], vraw[kHeads][2];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = sub + i * subs;
    kraw[i][0] = kraw[i][1] = vraw[i][0] = vraw[i][1] = make_uint2(0, 0);
    if (writing && h < heads) {
      kraw[i][0] = raw4(kr + h * p.k_head), kraw[i][1] = raw4(kr + h * p.k_head + 64);
      vraw[i][0] = raw4(vr + h * p.v_head), vraw[i][1] = raw4(vr + h * p.v_head + 64);
    }
  }
  float4 cl, ch, sl, sh;
  cl = ch = sl = sh = make_float4(0.f, 0.f, 0.f, 0.f);
  if (reading) {
    const float* c = cos + r * kCacheDim;
    const float* s = sin + r * kCacheDim;
    cl = *reinterpret_cast<const float4*>(c), ch = *reinterpret_cast<const float4*>(c + 64);
    sl = *reinterpret_cast<const float4*>(s), sh = *reinterpret_cast<const float4*>(s + 64);
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = sub + i * subs;
    if (i * subs >= heads) break;  // the same for the whole block: the shuffles below are the warp's
    const bool held = writing && h < heads;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float4 lo = widen<T>(which ? vraw[i][0] : kraw[i][0]), hi = widen<T>(which ? vraw[i][1] : kraw[i][1]);
      if (which == 0) rotate(lo, hi, cl, ch, sl, sh);
      bool bad = false;
      uint32_t top = take_finite(lo, bad);
      top = max(top, take_finite(hi, bad));
      if (bad && held) poisoned[h][which] = 1;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if ((threadIdx.x & 15) == 0 && held) atomicMax(&tops[h][which], top);
    }
  }
  // ---- queries, while the scales of the heads come together
  if (r < rows) {
    T* dst = out + (int64_t)r * p.H * kCacheDim;
    constexpr int kAhead = 4;
    for (int base = sub; base < heads * group; base += kAhead * subs) {
      uint2 w[kAhead][2];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int h = base + i * subs;
        w[i][0] = w[i][1] = make_uint2(0, 0);
        if (reading && h < heads * group) w[i][0] = raw4(qr + h * p.q_head), w[i][1] = raw4(qr + h * p.q_head + 64);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int h = base + i * subs;
        if (h >= heads * group) break;
        float4 lo = widen<T>(w[i][0]), hi = widen<T>(w[i][1]);
        rotate(lo, hi, cl, ch, sl, sh);
        store4(dst + h * kCacheDim, lo);
        store4(dst + h * kCacheDim + 64, hi);
      }
    }
  }
  if (writes == 0) return;
  __syncthreads();

  const int in_page = pos0 % p.page, off = pos0 % kCacheBlock;
  auto head_of = [&](int h, int which) { return ((int64_t)page * 2 + which) * p.KV + h0 + h; };
  // ---- a team settles a scale, and rounds the block's older tokens again if it grew
  if (team < 2 * heads) {
    const int h = team >> 1, which = team & 1;
    bool bad = poisoned[h][which] != 0;
    int e = scale_exponent(__uint_as_float(tops[h][which]));
    float* scale = p.scales + head_of(h, which) * (p.page / kCacheBlock) + in_page / kCacheBlock;
    if (off > 0) {
      const float was = *scale;
      if (!(fabsf(was) <= 3.402823466e38f)) {
        bad = true;
      } else {
        const int e_was = (__float_as_int(was) >> 23) - 127;
        if (e > e_was) {
          const float f = e - e_was < 127 ? two_to(e_was - e) : 0.f;
          uint2* b = reinterpret_cast<uint2*>(p.pages + (head_of(h, which) * p.page + in_page - off) * kCacheDim) + (threadIdx.x & 15);
#pragma unroll 4
          for (int r = 0; r < off; ++r) {
            const uint2 w = b[r * (kCacheDim / 8)];
            b[r * (kCacheDim / 8)] = make_uint2(to_e4m3(times(from_e4m3(w.x), f)), to_e4m3(times(from_e4m3(w.y), f)));
          }
        }
        e = max(e, e_was);
      }
    }
    __syncwarp(0xffffu << (threadIdx.x & 16));  // the team has read the old scale
    if ((threadIdx.x & 15) == 0) {
      exponents[h][which] = e;
      *scale = bad ? __int_as_float(0x7fc00000) : two_to(e);
    }
  }
  __syncthreads();
  // ---- bytes
  if (!writing) return;
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = sub + i * subs;
    if (h >= heads) break;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float4 lo = widen<T>(which ? vraw[i][0] : kraw[i][0]), hi = widen<T>(which ? vraw[i][1] : kraw[i][1]);
      if (which == 0) rotate(lo, hi, cl, ch, sl, sh);
      bool bad;
      take_finite(lo, bad), take_finite(hi, bad);
      const float inv = two_to(-exponents[h][which]);  // -120 <= -e <= 32
      uint8_t* b = p.pages + (head_of(h, which) * p.page + in_page + r) * kCacheDim + d;
      *reinterpret_cast<uint32_t*>(b) = to_e4m3(times(lo, inv));
      *reinterpret_cast<uint32_t*>(b + 64) = to_e4m3(times(hi, inv));
    }
  }
}

template <typename T>
cudaError_t launch_append(const AppendParams& p, cudaStream_t stream) {
  const dim3 grid(p.tokens / kCacheBlock + 3 * p.n + 1, (p.KV + kHeads - 1) / kHeads);
  return launch_after_previous(cache_append_kernel<T>, grid, kAppendThreads, 0, stream, p);
}

// ---------------------------------------------------------------------------------- pages
constexpr int kBook = 1024;        // threads of the bookkeeping block
constexpr int kMaxBatch = kBookBatch;
constexpr int kPer = 8;            // pages that one thread looks at in a step

// Exclusive sum of x over the block (kBook threads); `total` gets the sum.
__device__ __forceinline__ int block_scan(int x, int* warp_sums, int& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int v = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();  // the previous scan's sums have been read
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  total = warp_sums[kBook / 32 - 1];
  return v - x + (warp > 0 ? warp_sums[warp - 1] : 0);
}

// The first `want` free pages, lowest first, into found[]; returns how many there are (<= want).
// refs were written by other threads of this grid or of earlier kernels: read past L1.
__device__ int find_free(const int* refs, int npages, int want, int* found, int* warp_sums) {
  int have = 0;
  for (int base = 0; base < npages && have < want; base += kBook * kPer) {
    const int first = base + (int)threadIdx.x * kPer;
    int free_mask = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (first + i < npages && __ldcg(refs + first + i) == 0) free_mask |= 1 << i;
    int total;
    int rank = have + block_scan(__popc(free_mask), warp_sums, total);
    for (int m = free_mask; m && rank < want; m &= m - 1, ++rank) found[rank] = first + __ffs(m) - 1;
    have += total;
  }
  __syncthreads();
  return min(have, want);
}

__device__ __forceinline__ int last_not_above(const int* sums, int n, int x) {  // last i < n with sums[i] <= x
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sums[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Exclusive sums of need[0..n) in place (n <= kMaxBatch); returns the total.
__device__ int scan_needs(int* need, int n, int* warp_sums) {
  int sum = 0;
  for (int base = 0; base < n; base += kBook) {
    const int i = base + (int)threadIdx.x;
    const int x = i < n ? need[i] : 0;
    int total;
    const int before = block_scan(x, warp_sums, total);
    if (i < n) need[i] = sum + before;
    sum += total;
  }
  __syncthreads();
  return sum;
}

// Gives sequence i (slot seqs[i]) the pages for counts[i] more tokens, all or none of the batch.
// missing[0]: 0 done, > 0 pages that lack, -1 a slot, count or length that is not possible.
__global__ void __launch_bounds__(kBook) cache_reserve_kernel(int* table, int slots, int width, int* lens, int* refs,
                                                              int npages, const int* seqs, const int* counts, int n,
                                                              int page, int* found, int* missing) {
  __shared__ int need[kMaxBatch];
  __shared__ int warp_sums[32];
  __shared__ int bad, large;
  __shared__ int64_t sum;
  after_previous();
  if (threadIdx.x == 0) bad = large = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kBook) {
    const int slot = seqs[i], c = counts[i];
    int pages = 0;
    if (slot < 0 || slot >= slots || c < 0) {
      bad = 1;
    } else {
      const int len = lens[slot];
      const int64_t to = ((int64_t)len + c + page - 1) / page;
      if (len < 0 || to > width) bad = 1;
      else pages = (int)to - (len + page - 1) / page;
    }
    need[i] = pages;
    if (pages >= (int)((int64_t(1) << 31) / kMaxBatch)) large = 1;
  }
  __syncthreads();
  if (bad) {
    if (threadIdx.x == 0) *missing = -1;
    return;
  }
  if (large) {  // the sum may pass 32 bits: more than the pool has then
    if (threadIdx.x == 0) {
      sum = 0;
      for (int i = 0; i < n; ++i) sum += need[i];
    }
    __syncthreads();
    if (sum > npages) {
      const int have = find_free(refs, npages, npages, found, warp_sums);
      if (threadIdx.x == 0) *missing = (int)min(sum - have, (int64_t)0x7fffffff);
      return;
    }
  }
  const int total = scan_needs(need, n, warp_sums);
  const int have = find_free(refs, npages, min(total, npages), found, warp_sums);
  if (have < total) {
    if (threadIdx.x == 0) *missing = total - have;
    return;
  }
  for (int k = threadIdx.x; k < total; k += kBook) {
    const int i = last_not_above(need, n, k), slot = seqs[i];
    const int at = (lens[slot] + page - 1) / page + k - need[i];
    table[(int64_t)slot * width + at] = found[k];
    refs[found[k]] = 1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kBook) lens[seqs[i]] += counts[i];
  if (threadIdx.x == 0) *missing = 0;
}

// Takes slot seqs[blockIdx.x]'s pages from it.
__global__ void cache_free_kernel(int* table, int slots, int width, int* lens, int* refs, int npages, const int* seqs,
                                  int* status) {
  after_previous();
  const int slot = seqs[blockIdx.x];
  if (slot < 0 || slot >= slots) {
    if (threadIdx.x == 0) report(status, kCacheBadSlot);
    return;
  }
  for (int j = threadIdx.x; j < width; j += blockDim.x) {
    const int page = atomicExch(table + (int64_t)slot * width + j, -1);
    if (page >= npages) report(status, kCacheBadPage);
    else if (page >= 0) atomicSub(refs + page, 1);
  }
  if (threadIdx.x == 0) lens[slot] = 0;
}

// Slot dst[i] gives up its pages, takes those of src[i] that are full, and a free one for a last page
// that is not: the copy list from[i] -> to[i] (-1: nothing to copy, -2: a bad pair), lowest free page
// first in the order of the batch.  Where pages lack, every destination is left empty.
// One block: the entries of all pairs' rows are gone through by its threads, four ahead.
__global__ void __launch_bounds__(kBook) cache_fork_kernel(const Book b, const int* src, const int* dst, int n, int* from,
                                                           int* to, int* found, int* missing) {
  __shared__ int need[kMaxBatch];
  __shared__ int warp_sums[32];
  after_previous();
  const int64_t entries = (int64_t)n * b.width;
  auto good = [&](int s, int d) { return s >= 0 && s < b.slots && d >= 0 && d < b.slots && s != d; };
  for (int64_t base = threadIdx.x; base < entries; base += 4 * kBook) {
    int old[4], shared[4];
    int* entry[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int64_t k = base + x * kBook;
      old[x] = shared[x] = -1;
      entry[x] = nullptr;
      if (k >= entries) continue;
      const int i = (int)(k / b.width), j = (int)(k % b.width), s = src[i], d = dst[i];
      if (!good(s, d)) continue;
      entry[x] = b.table + (int64_t)d * b.width + j;
      old[x] = *entry[x];
      if (j < b.lens[s] / b.page) {
        shared[x] = b.table[(int64_t)s * b.width + j];
        if (shared[x] < 0 || shared[x] >= b.npages) {
          report(b.status, kCacheBadPage);
          shared[x] = -1;
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (entry[x] == nullptr) continue;
      *entry[x] = shared[x];
      if (shared[x] >= 0) atomicAdd(b.refs + shared[x], 1);
      if (old[x] >= b.npages) report(b.status, kCacheBadPage);
      else if (old[x] >= 0) atomicSub(b.refs + old[x], 1);
    }
  }
  for (int i = threadIdx.x; i < n; i += kBook) {
    const int s = src[i], d = dst[i];
    int last = -1;
    if (!good(s, d)) {
      report(b.status, kCacheBadSlot);
      last = -2;
    } else {
      if (b.lens[s] < 0) report(b.status, kCacheBadLength);  // read as none
      const int len = max(b.lens[s], 0), whole = len / b.page;
      if (len % b.page != 0) {
        last = whole < b.width ? b.table[(int64_t)s * b.width + whole] : -1;
        if (last < 0 || last >= b.npages) {
          report(b.status, kCacheBadPage);
          last = -1;
        }
      }
    }
    from[i] = last;
    need[i] = last >= 0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kBook)  // after every source length has been read
    if (from[i] != -2) b.lens[dst[i]] = max(b.lens[src[i]], 0);
  const int total = scan_needs(need, n, warp_sums);
  const int have = find_free(b.refs, b.npages, min(total, b.npages), found, warp_sums);
  const bool ok = have >= total;
  for (int i = threadIdx.x; i < n; i += kBook) {
    to[i] = -1;
    if (ok && from[i] >= 0) {
      const int fresh = found[need[i]], d = dst[i];
      to[i] = fresh;
      b.table[(int64_t)d * b.width + b.lens[d] / b.page] = fresh;
      b.refs[fresh] = 1;
    }
  }
  if (!ok) {
    __syncthreads();
    for (int64_t k = threadIdx.x; k < entries; k += kBook) {
      const int i = (int)(k / b.width);
      if (from[i] == -2) continue;
      int* entry = b.table + (int64_t)dst[i] * b.width + k % b.width;
      if (*entry >= 0) atomicSub(b.refs + *entry, 1);
      *entry = -1;
    }
    for (int i = threadIdx.x; i < n; i += kBook)
      if (from[i] != -2) b.lens[dst[i]] = 0;
  }
  if (threadIdx.x == 0) *missing = ok ? 0 : total - have;
}

// Where live pages go: those below `live` (their number) stay, the j-th live page from there on
// goes to the j-th free one below.  to[p] = -1 for a free page.  The counts go along: out_refs may
// be refs itself (a move in place), so they are kept in between.
__global__ void __launch_bounds__(kBook) cache_plan_kernel(const int* refs, int npages, int* out_refs, int room, int* holes,
                                                           int* to, int* kept, int* missing) {
  __shared__ int warp_sums[32];
  after_previous();
  int live = 0;
  for (int base = 0; base < npages; base += kBook * kPer) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int p = base + (int)threadIdx.x * kPer + i;
      if (p < npages) {
        const int count = refs[p];
        kept[p] = count;
        c += count != 0;
      }
    }
    int total;
    block_scan(c, warp_sums, total);
    live += total;
  }
  if (threadIdx.x == 0) *missing = max(live - room, 0);
  find_free(refs, min(live, npages), live, holes, warp_sums);
  int moved = 0;
  for (int base = 0; base < npages; base += kBook * kPer) {
    const int first = base + (int)threadIdx.x * kPer;
    int mask = 0, above = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int p = first + i;
      if (p < npages && kept[p] != 0) {
        mask |= 1 << i;
        if (p >= live) above |= 1 << i;
      }
    }
    int total;
    int rank = moved + block_scan(__popc(above), warp_sums, total);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int p = first + i;
      if (p < npages) to[p] = !(mask >> i & 1) ? -1 : (above >> i & 1) ? holes[rank++] : p;
    }
    moved += total;
  }
  if (live > room) return;
  __syncthreads();
  for (int p = threadIdx.x; p < room; p += kBook) out_refs[p] = 0;
  __syncthreads();
  for (int p = threadIdx.x; p < npages; p += kBook)
    if (to[p] >= 0) out_refs[to[p]] = kept[p];
}

// A block takes a whole page of a layer at a time, 32 KB in flight.
constexpr int kCopyThreads = 256;
constexpr int kCopyAhead = 8;

__device__ __forceinline__ bool copy_item(const CopyParams& p, int i, int& a, int& b) {
  a = p.from != nullptr ? p.from[i] : i;
  b = p.to[i];
  if (a < 0 || b < 0) return false;
  if (a >= p.npages || b >= p.out_npages) {
    if (threadIdx.x == 0) report(p.status, kCacheBadPage);
    return false;
  }
  return !(a == b && p.pages == p.out_pages);
}

// blockIdx.y: layers y, y + gridDim.y, ...; blockIdx.x: a share of the list.
__global__ void __launch_bounds__(kCopyThreads) cache_copy_kernel(const CopyParams p) {
  after_previous();
  if (p.missing != nullptr && *p.missing != 0) return;
  const int end = (int)(p.page_bytes / 16);
  for (int i = blockIdx.x; i < p.n; i += gridDim.x) {
    int a, b;
    if (!copy_item(p, i, a, b)) continue;
    for (int layer = blockIdx.y; layer < p.layers; layer += gridDim.y) {
      const int64_t in = layer * p.npages + a, out = layer * p.out_npages + b;
      const uint4* s = reinterpret_cast<const uint4*>(p.pages + in * p.page_bytes);
      uint4* o = reinterpret_cast<uint4*>(p.out_pages + out * p.page_bytes);
      for (int first = threadIdx.x; first < end; first += kCopyThreads * kCopyAhead) {
        uint4 v[kCopyAhead];
#pragma unroll
        for (int u = 0; u < kCopyAhead; ++u)
          if (first + u * kCopyThreads < end) v[u] = __ldcs(s + first + u * kCopyThreads);
#pragma unroll
        for (int u = 0; u < kCopyAhead; ++u)
          if (first + u * kCopyThreads < end) __stcs(o + first + u * kCopyThreads, v[u]);
      }
      for (int f = threadIdx.x; f < p.scale_floats; f += kCopyThreads)
        p.out_scales[out * p.scale_floats + f] = p.scales[in * p.scale_floats + f];
    }
  }
  if (p.out_table != nullptr) {
    const int64_t block = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, blocks = (int64_t)gridDim.x * gridDim.y;
    for (int64_t k = block * kCopyThreads + threadIdx.x; k < p.entries; k += blocks * kCopyThreads) {
      const int page = p.table[k];
      int to = -1;
      if (page >= p.npages) report(p.status, kCacheBadPage);
      else if (page >= 0) to = p.to[page];
      p.out_table[k] = to;
    }
  }
}

}  // namespace

namespace mimir {

cudaError_t cache_status_address(void** word) { return cudaGetSymbolAddress(word, g_cache_status); }

cudaError_t launch_cache_append(const AppendParams& p, bool bf16, cudaStream_t stream) {
  return bf16 ? launch_append<__nv_bfloat16>(p, stream) : launch_append<__half>(p, stream);
}

cudaError_t launch_cache_reserve(const Book& b, const int* seqs, const int* counts, int n, int* found, int* missing,
                                 cudaStream_t stream) {
  return launch_after_previous(cache_reserve_kernel, 1, kBook, 0, stream, b.table, b.slots, b.width, b.lens, b.refs, b.npages,
                               seqs, counts, n, b.page, found, missing);
}

cudaError_t launch_cache_free(const Book& b, const int* seqs, int n, cudaStream_t stream) {
  return launch_after_previous(cache_free_kernel, n, 256, 0, stream, b.table, b.slots, b.width, b.lens, b.refs, b.npages, seqs,
                               b.status);
}

cudaError_t launch_cache_fork(const Book& b, const int* src, const int* dst, int n, int* from, int* to, int* found,
                              int* missing, cudaStream_t stream) {
  return launch_after_previous(cache_fork_kernel, 1, kBook, 0, stream, b, src, dst, n, from, to, found, missing);
}

cudaError_t launch_cache_plan(const int* refs, int npages, int* out_refs, int room, int* holes, int* to, int* kept,
                              int* missing, cudaStream_t stream) {
  return launch_after_previous(cache_plan_kernel, 1, kBook, 0, stream, refs, npages, out_refs, room, holes, to, kept, missing);
}

cudaError_t launch_cache_copy(const CopyParams& p, cudaStream_t stream) {
  if (p.layers == 0 || (p.n == 0 && p.entries == 0)) return cudaSuccess;
  const int y = std::min(p.layers, 65535);
  const int x = std::min(std::max(p.n, 1), std::max(1, 148 * 8 / y));
  return launch_after_previous(cache_copy_kernel, dim3(x, y), kCopyThreads, 0, stream, p);
}

}  // namespace mimir
