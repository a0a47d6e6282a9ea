// The 8-bit paged key/value cache: rotary + quantise + write (cache_append), and the bookkeeping
// and movement of its pages (cache_reserve, cache_free, cache_fork, cache_compact, cache_copy).
// Layout and status codes: kv_cache.cuh.
//
// Append.  A new token at position p gets x' = x * cos[p] + rot(x) * sin[p] (k and q; the two
// products and their sum each rounded to fp32) and v' = v.  All new tokens of one head in one
// block of 16 share the scale 2^e with e the smallest exponent (>= -32) such that no |x'| is over
// 448 * 2^e, and not below the exponent of the tokens that the block already holds; where those
// held a smaller one, their bytes are rounded again to the new one.  Powers of two make every
// product and quotient with a scale exact, so a value is rounded once (e4m3, nearest even), and
// a token whose block later grows is rounded again only where it falls below the normal range.
// One warp owns a (block, head, k or v): two tokens at a time, 16 lanes a token, each lane four
// dimensions of either half, so that both partners of a rotation are in one thread and all
// loads are 8 bytes a lane; the whole block stays in registers between the maximum and the write.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "kv_cache.cuh"

using namespace mimir;

namespace {

__device__ int g_cache_status;

__device__ __forceinline__ void report(int* status, int code) { atomicCAS(status, 0, code); }

__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 load4(const __half* p) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
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

// Rotates dimensions d..d+3 (lo) and d+64..d+67 (hi) of one head.
__device__ __forceinline__ void rotate(float4& lo, float4& hi, const float* cos_row, const float* sin_row, int d) {
  const float4 cl = *reinterpret_cast<const float4*>(cos_row + d), ch = *reinterpret_cast<const float4*>(cos_row + 64 + d);
  const float4 sl = *reinterpret_cast<const float4*>(sin_row + d), sh = *reinterpret_cast<const float4*>(sin_row + 64 + d);
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

// A value that is not finite becomes zero and is reported in `bad`.
__device__ __forceinline__ void take_finite(float4& v, float& amax, bool& bad) {
  float* x = reinterpret_cast<float*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!(fabsf(x[i]) <= 3.402823466e38f)) {
      x[i] = 0.f;
      bad = true;
    }
    amax = fmaxf(amax, fabsf(x[i]));
  }
}

constexpr int kAppendThreads = 256;
constexpr int kMaxChunk = 16;

template <typename T>
struct AppendParams {
  const T *q, *k, *v;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;  // strides in elements
  T* q_out;                                             // [tokens, H, 128]
  const float *cos, *sin;
  int64_t positions;
  uint8_t* pages;
  float* scales;
  int64_t npages;
  const int *table, *lens, *seqs, *cu;
  int slots, width, n, tokens, H, KV, page, chunk;
  int* status;
};

struct TokenInfo {
  int pos;     // -1: no position (the row belongs to no sequence, or its slot or length is bad)
  int page;    // -1: nothing is written
  int count;   // tokens of its block that it leads (0: another token leads)
};

// blockIdx.x: `chunk` rows of the new tokens; blockIdx.y: a key/value head and its query heads.
template <typename T>
__global__ void __launch_bounds__(kAppendThreads) cache_append_kernel(const AppendParams<T> p) {
  __shared__ TokenInfo info[kMaxChunk];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = blockIdx.x * p.chunk;
  const int here = min(p.chunk, p.tokens - t0);
  for (int r = warp; r < here; r += kAppendThreads / 32) {
    const int t = t0 + r;
    // the last i with cu[i] <= t, 32 candidates a step
    int lo = 0, size = p.n + 1;
    while (size > 1) {
      const int step = (size + 31) / 32;
      const int at = lo + lane * step;
      const int c = __popc(__ballot_sync(0xffffffffu, at < lo + size && p.cu[min(at, p.n)] <= t));
      const int next = lo + max(c - 1, 0) * step;
      size = min(step, lo + size - next);
      lo = next;
    }
    if (lane == 0) {
      TokenInfo ti{-1, -1, 0};
      if (lo < p.n) {
        const int first = p.cu[lo], end = min(p.cu[lo + 1], p.tokens), slot = p.seqs[lo];
        if (t < first || slot < 0 || slot >= p.slots) {
          report(p.status, kCacheBadSlot);
        } else {
          const int start = p.lens[slot] - (p.cu[lo + 1] - first);
          const int pos = start + t - first;
          if (start < 0 || pos >= p.positions) {
            report(p.status, kCacheBadLength);
          } else {
            ti.pos = pos;
            const int j = pos / p.page;
            const int page = j < p.width ? p.table[(int64_t)slot * p.width + j] : -1;
            if (page < 0 || page >= p.npages) report(p.status, kCacheBadPage);
            else ti.page = page;
            if (t == first || pos % kCacheBlock == 0)
              ti.count = min(min(kCacheBlock - pos % kCacheBlock, end - t), (int)p.positions - pos);
          }
        }
      }
      info[r] = ti;
    }
  }
  __syncthreads();

  const int kvh = blockIdx.y, group = p.H / p.KV;
  const int half = lane >> 4, d = (lane & 15) * 4;
  // ---- keys and values: item 2r is the keys of the block that row r leads, 2r + 1 its values
  for (int item = warp; item < 2 * here; item += kAppendThreads / 32) {
    const TokenInfo ti = info[item >> 1];
    if (ti.count == 0 || ti.page < 0) continue;
    const bool is_v = item & 1;
    const int t = t0 + (item >> 1);
    const T* src = is_v ? p.v + kvh * p.v_head : p.k + kvh * p.k_head;
    const int64_t tok = is_v ? p.v_tok : p.k_tok;
    float4 lo[8], hi[8];
    float amax = 0.f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 2 * i + half;
      lo[i] = hi[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < ti.count) {
        lo[i] = load4(src + (t + r) * tok + d);
        hi[i] = load4(src + (t + r) * tok + 64 + d);
      }
    }
    if (!is_v) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 2 * i + half;
        if (r < ti.count) {
          const int64_t row = (int64_t)(ti.pos + r) * kCacheDim;
          rotate(lo[i], hi[i], p.cos + row, p.sin + row, d);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      take_finite(lo[i], amax, bad);
      take_finite(hi[i], amax, bad);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    bad = __any_sync(0xffffffffu, bad);

    const int in_page = ti.pos % p.page, off = ti.pos % kCacheBlock;
    const int64_t head = ((int64_t)ti.page * 2 + (is_v ? 1 : 0)) * p.KV + kvh;
    float* scale = p.scales + head * (p.page / kCacheBlock) + in_page / kCacheBlock;
    uint8_t* base = p.pages + (head * p.page + (in_page - off)) * kCacheDim;  // the block's first token
    int e = scale_exponent(amax);
    if (off > 0) {
      const float was = *scale;
      if (!(fabsf(was) <= 3.402823466e38f)) {
        bad = true;
      } else {
        const int e_was = (__float_as_int(was) >> 23) - 127;
        if (e > e_was) {  // older tokens are rounded again
          const float f = e - e_was < 127 ? two_to(e_was - e) : 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = 2 * i + half;
            if (r < off) {
              uint2* b = reinterpret_cast<uint2*>(base + r * kCacheDim) + (lane & 15);
              const uint2 w = *b;
              *b = make_uint2(to_e4m3(times(from_e4m3(w.x), f)), to_e4m3(times(from_e4m3(w.y), f)));
            }
          }
        }
        e = max(e, e_was);
      }
    }
    const float inv = two_to(-e);  // -120 <= -e <= 32
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 2 * i + half;
      if (r < ti.count) {
        uint8_t* b = base + (off + r) * kCacheDim + d;
        *reinterpret_cast<uint32_t*>(b) = to_e4m3(times(lo[i], inv));
        *reinterpret_cast<uint32_t*>(b + 64) = to_e4m3(times(hi[i], inv));
      }
    }
    __syncwarp();  // every lane has read the old scale
    if (lane == 0) *scale = bad ? __int_as_float(0x7fc00000) : two_to(e);
  }
  // ---- queries: two rows (token, head of the group) a warp
  for (int item = warp * 2 + half; item < here * group; item += kAppendThreads / 16) {
    const int r = item / group, h = kvh * group + item % group;
    const TokenInfo ti = info[r];
    float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
    if (ti.pos >= 0) {
      const T* src = p.q + (t0 + r) * p.q_tok + h * p.q_head;
      lo = load4(src + d);
      hi = load4(src + 64 + d);
      const int64_t row = (int64_t)ti.pos * kCacheDim;
      rotate(lo, hi, p.cos + row, p.sin + row, d);
    }
    T* dst = p.q_out + ((int64_t)(t0 + r) * p.H + h) * kCacheDim;
    store4(dst + d, lo);
    store4(dst + 64 + d, hi);
  }
}

template <typename T>
void launch_append(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& cos,
                   const at::Tensor& sin, const at::Tensor& pages, const at::Tensor& scales, const at::Tensor& table,
                   const at::Tensor& lens, const at::Tensor& seqs, const at::Tensor& cu, at::Tensor& out) {
  AppendParams<T> p{};
  p.q = reinterpret_cast<const T*>(q.data_ptr());
  p.k = reinterpret_cast<const T*>(k.data_ptr());
  p.v = reinterpret_cast<const T*>(v.data_ptr());
  p.q_tok = q.stride(0), p.q_head = q.stride(1);
  p.k_tok = k.stride(0), p.k_head = k.stride(1);
  p.v_tok = v.stride(0), p.v_head = v.stride(1);
  p.q_out = reinterpret_cast<T*>(out.data_ptr());
  p.cos = cos.data_ptr<float>(), p.sin = sin.data_ptr<float>();
  p.positions = cos.size(0);
  p.pages = reinterpret_cast<uint8_t*>(pages.data_ptr());
  p.scales = scales.data_ptr<float>();
  p.npages = pages.size(0);
  p.table = table.data_ptr<int>(), p.lens = lens.data_ptr<int>();
  p.seqs = seqs.data_ptr<int>(), p.cu = cu.data_ptr<int>();
  p.slots = (int)table.size(0), p.width = (int)table.size(1), p.n = (int)seqs.size(0);
  p.tokens = (int)q.size(0), p.H = (int)q.size(1), p.KV = (int)k.size(1), p.page = (int)pages.size(3);
  // Few tokens: more and smaller blocks, so that every block of 16 tokens has a warp at once.
  p.chunk = p.tokens >= 2048 ? kMaxChunk : 4;
  p.status = cache_status_word(q.device());
  const dim3 grid((unsigned)((p.tokens + p.chunk - 1) / p.chunk), (unsigned)p.KV);
  cache_append_kernel<T><<<grid, kAppendThreads, 0, at::cuda::getCurrentCUDAStream()>>>(p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// ---------------------------------------------------------------------------------- pages
constexpr int kBook = 1024;        // threads of the bookkeeping block
constexpr int kMaxBatch = 4096;    // sequences of one call
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
  __shared__ int bad;
  if (threadIdx.x == 0) bad = 0;
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
  }
  __syncthreads();
  if (bad) {
    if (threadIdx.x == 0) *missing = -1;
    return;
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

// Slot dst[i] gives up its pages and takes those of src[i] that are full; part[i] = the page that
// has to be copied, or -1.
__global__ void cache_share_kernel(int* table, int slots, int width, int* lens, int* refs, int npages, const int* src,
                                   const int* dst, int page, int* part, int* status) {
  const int i = blockIdx.x, a = src[i], b = dst[i];
  if (a < 0 || a >= slots || b < 0 || b >= slots || a == b) {
    if (threadIdx.x == 0) {
      report(status, kCacheBadSlot);
      part[i] = -2;
    }
    return;
  }
  const int len = lens[a], whole = min(len / page, width);
  for (int j = threadIdx.x; j < width; j += blockDim.x) {
    const int old = atomicExch(table + (int64_t)b * width + j, -1);
    if (old >= npages) report(status, kCacheBadPage);
    else if (old >= 0) atomicSub(refs + old, 1);
    if (j < whole) {
      const int shared = table[(int64_t)a * width + j];
      if (shared < 0 || shared >= npages) {
        report(status, kCacheBadPage);
      } else {
        table[(int64_t)b * width + j] = shared;
        atomicAdd(refs + shared, 1);
      }
    }
  }
  if (threadIdx.x == 0) {
    lens[b] = len;
    int last = -1;
    if (len % page != 0) {
      last = whole < width ? table[(int64_t)a * width + whole] : -1;
      if (last < 0 || last >= npages) {
        report(status, kCacheBadPage);
        last = -1;
      }
    }
    part[i] = last;
  }
}

// Fresh pages for the partly filled ones: copy lists from[i] -> to[i] (-1: nothing), lowest free
// page first in the order of the batch.  Where pages lack, every destination is left empty.
__global__ void __launch_bounds__(kBook) cache_fork_kernel(int* table, int width, int* lens, int* refs, int npages,
                                                           const int* dst, int n, int page, int* from, int* to,
                                                           int* found, int* missing) {
  __shared__ int need[kMaxBatch];
  __shared__ int warp_sums[32];
  for (int i = threadIdx.x; i < n; i += kBook) need[i] = from[i] >= 0;
  __syncthreads();
  const int total = scan_needs(need, n, warp_sums);
  const int have = find_free(refs, npages, min(total, npages), found, warp_sums);
  const bool ok = have >= total;
  for (int i = threadIdx.x; i < n; i += kBook) {
    const bool mine = from[i] >= 0;
    to[i] = -1;
    if (ok && mine) {
      const int fresh = found[need[i]], b = dst[i];
      to[i] = fresh;
      table[(int64_t)b * width + lens[b] / page] = fresh;
      refs[fresh] = 1;
    }
  }
  if (!ok) {
    __syncthreads();
    for (int64_t k = threadIdx.x; k < (int64_t)n * width; k += kBook) {
      const int i = (int)(k / width);
      if (from[i] == -2) continue;
      int* entry = table + (int64_t)dst[i] * width + k % width;
      const int old = *entry;
      if (old >= 0 && old < npages) atomicSub(refs + old, 1);
      *entry = -1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kBook)
      if (from[i] != -2) lens[dst[i]] = 0;
  }
  if (threadIdx.x == 0) *missing = ok ? 0 : total - have;
}

// Where live pages go: those below `live` (their number) stay, the j-th live page from there on
// goes to the j-th free one below.  to[p] = -1 for a free page.
__global__ void __launch_bounds__(kBook) cache_plan_kernel(const int* refs, int npages, int room, int* holes, int* to,
                                                           int* missing) {
  __shared__ int warp_sums[32];
  int live = 0;
  for (int base = 0; base < npages; base += kBook * kPer) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int p = base + (int)threadIdx.x * kPer + i;
      c += p < npages && refs[p] != 0;
    }
    int total;
    block_scan(c, warp_sums, total);
    live += total;
  }
  if (threadIdx.x == 0) *missing = max(live - room, 0);
  find_free(refs, live, live, holes, warp_sums);
  int moved = 0;
  for (int base = 0; base < npages; base += kBook * kPer) {
    const int first = base + (int)threadIdx.x * kPer;
    int mask = 0, above = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int p = first + i;
      if (p < npages && refs[p] != 0) {
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
}

constexpr int kCopyThreads = 256;
constexpr int kCopyBytes = kCopyThreads * 16 * 4;  // one block's share of a page in a step

// Copies page from[i] of every layer to page to[i] (i itself where `from` is null; nothing where
// either is negative or both are the same page of one pool), bytes and scales.
struct CopyParams {
  const uint8_t* pages;
  const float* scales;
  uint8_t* out_pages;
  float* out_scales;
  int64_t npages, out_npages;
  int64_t page_bytes;
  int scale_floats, layers, n;
  const int *from, *to, *missing;
  int* status;
  // compaction: the table and the counts of the new pool
  const int *table, *refs;
  int *out_table, *out_refs;
  int64_t entries;
};

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

__global__ void __launch_bounds__(kCopyThreads) cache_copy_kernel(const CopyParams p) {
  if (p.missing != nullptr && *p.missing != 0) return;
  const int64_t parts = (p.page_bytes + kCopyBytes - 1) / kCopyBytes;
  const int64_t total = parts * p.n * p.layers;
  for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
    const int64_t part = w % parts, rest = w / parts;
    const int i = (int)(rest % p.n);
    const int64_t layer = rest / p.n;
    int a, b;
    if (!copy_item(p, i, a, b)) continue;
    const int64_t in = layer * p.npages + a, out = layer * p.out_npages + b;
    const uint4* s = reinterpret_cast<const uint4*>(p.pages + in * p.page_bytes);
    uint4* o = reinterpret_cast<uint4*>(p.out_pages + out * p.page_bytes);
    const int64_t end = p.page_bytes / 16, first = part * (kCopyBytes / 16) + threadIdx.x;
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (first + u * kCopyThreads < end) v[u] = s[first + u * kCopyThreads];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (first + u * kCopyThreads < end) o[first + u * kCopyThreads] = v[u];
    if (part == 0)
      for (int f = threadIdx.x; f < p.scale_floats; f += kCopyThreads)
        p.out_scales[out * p.scale_floats + f] = p.scales[in * p.scale_floats + f];
  }
  if (p.out_table != nullptr) {
    for (int64_t k = blockIdx.x * (int64_t)kCopyThreads + threadIdx.x; k < p.entries; k += (int64_t)gridDim.x * kCopyThreads) {
      const int page = p.table[k];
      int to = -1;
      if (page >= p.npages) report(p.status, kCacheBadPage);
      else if (page >= 0) to = p.to[page];
      p.out_table[k] = to;
    }
  }
}

// Counts of a compacted pool: page to[p] of the new pool has the count of page p, the rest are free.
__global__ void cache_counts_kernel(const int* refs, const int* to, int npages, int* out_refs, const int* missing) {
  if (*missing != 0) return;
  for (int p = blockIdx.x * blockDim.x + threadIdx.x; p < npages; p += gridDim.x * blockDim.x)
    if (to[p] >= 0) out_refs[to[p]] = refs[p];
}
__global__ void cache_zero_counts_kernel(int* out_refs, int n, const int* missing) {
  if (*missing != 0) return;
  for (int p = blockIdx.x * blockDim.x + threadIdx.x; p < n; p += gridDim.x * blockDim.x) out_refs[p] = 0;
}

void launch_copy(CopyParams p, const at::Tensor& pages) {
  p.page_bytes = pages.size(2) * pages.size(3) * pages.size(4) * pages.size(5);
  p.scale_floats = (int)(p.page_bytes / kCacheDim / kCacheBlock);
  p.layers = (int)pages.size(0);
  p.npages = pages.size(1);
  const int64_t parts = (p.page_bytes + kCopyBytes - 1) / kCopyBytes * p.n * p.layers;
  const int64_t work = std::max<int64_t>(parts, p.out_table != nullptr ? (p.entries + kCopyThreads - 1) / kCopyThreads : 0);
  if (work == 0) return;
  cache_copy_kernel<<<(unsigned)std::min<int64_t>(work, 148 * 8), kCopyThreads, 0, at::cuda::getCurrentCUDAStream()>>>(p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void check_book(const at::Tensor& table, const at::Tensor& lens, const at::Tensor& refs) {
  CACHE_CHECK(table.is_cuda(), "page_table must be a CUDA tensor");
  check_int32(table, "page_table", 2, table.device());
  check_int32(lens, "seq_lens", 1, table.device());
  check_int32(refs, "ref_counts", 1, table.device());
  CACHE_CHECK(lens.size(0) == table.size(0), "seq_lens needs one length for each row of page_table");
  CACHE_CHECK(refs.size(0) < (int64_t(1) << 30), "the pool has too many pages");
}

void check_page_size(int64_t page) {
  CACHE_CHECK(page >= 16 && page <= 256 && (page & (page - 1)) == 0, "page_size must be 16, 32, 64, 128 or 256, not ",
              page);
}

}  // namespace

namespace mimir {
int* cache_status_word(const at::Device& dev) {
  static int* words[64] = {nullptr};
  const int i = dev.index();
  if (words[i] == nullptr) {
    c10::cuda::CUDAGuard guard(dev);
    void* ptr = nullptr;
    C10_CUDA_CHECK(cudaGetSymbolAddress(&ptr, g_cache_status));
    words[i] = reinterpret_cast<int*>(ptr);
  }
  return words[i];
}
}  // namespace mimir

// The first status code of a cache kernel since the last read (0: none).
int64_t cache_status(int64_t device) {
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
  int* word = cache_status_word(at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(device)));
  int host = 0;
  C10_CUDA_CHECK(cudaStreamSynchronize(at::cuda::getCurrentCUDAStream()));  // this stream's kernels have reported
  C10_CUDA_CHECK(cudaMemcpy(&host, word, sizeof(int), cudaMemcpyDeviceToHost));
  if (host) C10_CUDA_CHECK(cudaMemset(word, 0, sizeof(int)));
  return host;
}

at::Tensor cache_append(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor cos, at::Tensor sin, at::Tensor pages,
                        at::Tensor scales, at::Tensor table, at::Tensor lens, at::Tensor seqs, at::Tensor cu_new) {
  check_pool(pages, scales, 0);
  const at::Device dev = pages.device();
  check_rows(q, "q", dev);
  check_rows(k, "k", dev);
  check_rows(v, "v", dev);
  check_batch(table, lens, seqs, cu_new, dev);
  CACHE_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(), "q, k and v must have one type");
  CACHE_CHECK(k.size(1) == pages.size(2) && v.size(1) == pages.size(2), "k and v must have the pages' ", pages.size(2),
              " heads");
  CACHE_CHECK(k.size(0) == q.size(0) && v.size(0) == q.size(0), "q, k and v must have as many tokens");
  CACHE_CHECK(q.size(1) >= 1 && q.size(1) % k.size(1) == 0, "query heads ", q.size(1),
              " must be divisible by key/value heads ", k.size(1));
  for (const at::Tensor* t : {&cos, &sin})
    CACHE_CHECK(t->device() == dev && t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(1) == kCacheDim &&
                    t->is_contiguous() && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                "cos and sin must be contiguous float32 tables [positions, 128]");
  CACHE_CHECK(cos.size(0) == sin.size(0), "cos and sin must have as many positions");
  CACHE_CHECK(q.size(0) < (int64_t(1) << 31) - 64 && k.size(1) < 65536, "too many tokens or heads");
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor out = at::empty({q.size(0), q.size(1), kCacheDim}, q.options());
  if (q.size(0) == 0) return out;
  if (q.scalar_type() == at::kBFloat16)
    launch_append<__nv_bfloat16>(q, k, v, cos, sin, pages, scales, table, lens, seqs, cu_new, out);
  else
    launch_append<__half>(q, k, v, cos, sin, pages, scales, table, lens, seqs, cu_new, out);
  return out;
}

at::Tensor cache_reserve(at::Tensor table, at::Tensor lens, at::Tensor refs, at::Tensor seqs, at::Tensor counts,
                         int64_t page) {
  check_book(table, lens, refs);
  check_int32(seqs, "seqs", 1, table.device());
  check_int32(counts, "counts", 1, table.device());
  check_page_size(page);
  const int64_t n = seqs.size(0);
  CACHE_CHECK(counts.size(0) == n, "counts needs one entry for each of seqs");
  CACHE_CHECK(n <= kMaxBatch, "at most ", kMaxBatch, " sequences a call");
  c10::cuda::CUDAGuard guard(table.device());
  // [missing | free pages found]
  const int64_t most = std::min<int64_t>(n * table.size(1), refs.size(0));
  at::Tensor work = at::empty({1 + std::max<int64_t>(most, 1)}, refs.options());
  int* w = work.data_ptr<int>();
  cache_reserve_kernel<<<1, kBook, 0, at::cuda::getCurrentCUDAStream()>>>(
      table.data_ptr<int>(), (int)table.size(0), (int)table.size(1), lens.data_ptr<int>(), refs.data_ptr<int>(),
      (int)refs.size(0), seqs.data_ptr<int>(), counts.data_ptr<int>(), (int)n, (int)page, w + 1, w);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return work.narrow(0, 0, 1);
}

void cache_free(at::Tensor table, at::Tensor lens, at::Tensor refs, at::Tensor seqs) {
  check_book(table, lens, refs);
  check_int32(seqs, "seqs", 1, table.device());
  if (seqs.size(0) == 0) return;
  c10::cuda::CUDAGuard guard(table.device());
  cache_free_kernel<<<(unsigned)seqs.size(0), 256, 0, at::cuda::getCurrentCUDAStream()>>>(
      table.data_ptr<int>(), (int)table.size(0), (int)table.size(1), lens.data_ptr<int>(), refs.data_ptr<int>(),
      (int)refs.size(0), seqs.data_ptr<int>(), cache_status_word(table.device()));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

at::Tensor cache_fork(at::Tensor pages, at::Tensor scales, at::Tensor table, at::Tensor lens, at::Tensor refs,
                      at::Tensor src, at::Tensor dst) {
  check_pool(pages, scales, 1);
  check_book(table, lens, refs);
  CACHE_CHECK(table.device() == pages.device(), "page_table and pages must be on one device");
  check_int32(src, "src", 1, table.device());
  check_int32(dst, "dst", 1, table.device());
  CACHE_CHECK(refs.size(0) == pages.size(1), "ref_counts needs one count for each page");
  const int64_t n = src.size(0);
  CACHE_CHECK(dst.size(0) == n, "src and dst must have as many slots");
  CACHE_CHECK(n <= kMaxBatch, "at most ", kMaxBatch, " sequences a call");
  c10::cuda::CUDAGuard guard(table.device());
  at::Tensor work = at::empty({1 + 3 * std::max<int64_t>(n, 1)}, refs.options());  // missing | from | to | found
  int* w = work.data_ptr<int>();
  const int page = (int)pages.size(4), width = (int)table.size(1), np = (int)refs.size(0);
  auto st = at::cuda::getCurrentCUDAStream();
  if (n > 0) {
    cache_share_kernel<<<(unsigned)n, 256, 0, st>>>(table.data_ptr<int>(), (int)table.size(0), width, lens.data_ptr<int>(),
                                                    refs.data_ptr<int>(), np, src.data_ptr<int>(), dst.data_ptr<int>(),
                                                    page, w + 1, cache_status_word(table.device()));
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  cache_fork_kernel<<<1, kBook, 0, st>>>(table.data_ptr<int>(), width, lens.data_ptr<int>(), refs.data_ptr<int>(), np,
                                         dst.data_ptr<int>(), (int)n, page, w + 1, w + 1 + n, w + 1 + 2 * n, w);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (n > 0) {
    CopyParams p{};
    p.pages = reinterpret_cast<const uint8_t*>(pages.data_ptr());
    p.out_pages = reinterpret_cast<uint8_t*>(pages.data_ptr());
    p.scales = scales.data_ptr<float>();
    p.out_scales = scales.data_ptr<float>();
    p.out_npages = pages.size(1);
    p.n = (int)n;
    p.from = w + 1;
    p.to = w + 1 + n;
    p.missing = w;
    p.status = cache_status_word(table.device());
    launch_copy(p, pages);
  }
  return work.narrow(0, 0, 1);
}

void cache_copy(at::Tensor pages, at::Tensor scales, at::Tensor src, at::Tensor dst) {
  check_pool(pages, scales, 1);
  check_int32(src, "src", 1, pages.device());
  check_int32(dst, "dst", 1, pages.device());
  CACHE_CHECK(src.size(0) == dst.size(0), "src and dst must have as many pages");
  c10::cuda::CUDAGuard guard(pages.device());
  CopyParams p{};
  p.pages = reinterpret_cast<const uint8_t*>(pages.data_ptr());
  p.out_pages = reinterpret_cast<uint8_t*>(pages.data_ptr());
  p.scales = scales.data_ptr<float>();
  p.out_scales = scales.data_ptr<float>();
  p.out_npages = pages.size(1);
  p.n = (int)src.size(0);
  p.from = src.data_ptr<int>();
  p.to = dst.data_ptr<int>();
  p.status = cache_status_word(pages.device());
  launch_copy(p, pages);
}

// out_*: another pool (its table the shape of `table`), or the same tensors for a move in place.
at::Tensor cache_compact(at::Tensor pages, at::Tensor scales, at::Tensor table, at::Tensor refs, at::Tensor out_pages,
                         at::Tensor out_scales, at::Tensor out_table, at::Tensor out_refs) {
  check_pool(pages, scales, 1);
  check_pool(out_pages, out_scales, 1);
  const at::Device dev = pages.device();
  check_int32(table, "page_table", 2, dev);
  check_int32(refs, "ref_counts", 1, dev);
  check_int32(out_table, "the new page_table", 2, dev);
  check_int32(out_refs, "the new ref_counts", 1, dev);
  CACHE_CHECK(out_pages.device() == dev, "both pools must be on one device");
  CACHE_CHECK(out_table.sizes() == table.sizes(), "the new page_table must have the shape of the old one");
  CACHE_CHECK(refs.size(0) == pages.size(1) && out_refs.size(0) == out_pages.size(1),
              "ref_counts needs one count for each page");
  for (int64_t i : {0, 2, 3, 4, 5})
    CACHE_CHECK(pages.size(i) == out_pages.size(i), "the new pool must differ in its number of pages only");
  const bool in_place = pages.data_ptr() == out_pages.data_ptr();
  CACHE_CHECK(in_place == (table.data_ptr() == out_table.data_ptr()) && in_place == (refs.data_ptr() == out_refs.data_ptr()) &&
                  in_place == (scales.data_ptr() == out_scales.data_ptr()) &&
                  (!in_place || pages.size(1) == out_pages.size(1)),
              "compact into a pool of its own, or in place throughout");
  c10::cuda::CUDAGuard guard(dev);
  const int np = (int)refs.size(0);
  at::Tensor work = at::empty({1 + 3 * (int64_t)std::max(np, 1)}, refs.options());  // missing | to | holes | old counts
  int* w = work.data_ptr<int>();
  auto st = at::cuda::getCurrentCUDAStream();
  cache_plan_kernel<<<1, kBook, 0, st>>>(refs.data_ptr<int>(), np, (int)out_refs.size(0), w + 1 + np, w + 1, w);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  const int* counts = refs.data_ptr<int>();
  if (in_place && np > 0) {
    int* kept = w + 1 + 2 * (int64_t)np;
    C10_CUDA_CHECK(cudaMemcpyAsync(kept, counts, sizeof(int) * np, cudaMemcpyDeviceToDevice, st));
    counts = kept;
  }
  const int on = (int)out_refs.size(0);
  if (on > 0) cache_zero_counts_kernel<<<std::min(148, (on + 255) / 256), 256, 0, st>>>(out_refs.data_ptr<int>(), on, w);
  if (np > 0) cache_counts_kernel<<<std::min(148, (np + 255) / 256), 256, 0, st>>>(counts, w + 1, np, out_refs.data_ptr<int>(), w);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  CopyParams p{};
  p.pages = reinterpret_cast<const uint8_t*>(pages.data_ptr());
  p.out_pages = reinterpret_cast<uint8_t*>(out_pages.data_ptr());
  p.scales = scales.data_ptr<float>();
  p.out_scales = out_scales.data_ptr<float>();
  p.out_npages = out_pages.size(1);
  p.n = np;
  p.to = w + 1;
  p.missing = w;
  p.status = cache_status_word(dev);
  p.table = table.data_ptr<int>();
  p.out_table = out_table.data_ptr<int>();
  p.entries = table.numel();
  launch_copy(p, pages);
  return work.narrow(0, 0, 1);
}
