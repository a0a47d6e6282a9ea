// Penalties, biases and grammar masks on the logits of the next token, one pass over them.
//
//   x = logits[b, v]
//   v among the row's tokens:                x = x > 0 ? x / repetition[b] : x * repetition[b]
//   c > 0 of the generated tokens are v:     x = x - frequency[b] * c - presence[b]
//   x = x + the row's biases for v
//   v not allowed:                           x = -inf
//
// in fp32.  A block owns a slice of one row's vocabulary.  A few blocks an SM wait for memory most of
// their time, so a block asks for all that it can at once: its logits, the row's first 4096 tokens
// before it knows how many count, the biases before it knows which are its own.  It counts the row's tokens that fall into its slice in shared memory (whole numbers,
// so the order of the atomics does not matter); the few biases of the slice lie in a list, equal ids
// summed in their order, and a token's word says which of them is its own.  The history is read by every block of a row, from L2 after the first, so slices are large.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "serving.h"

using namespace mimir;

namespace {

constexpr int kThreads = 512;
constexpr int kSlice = 8192;               // 32 KB of counts
constexpr int kEach = kSlice / kThreads;   // logits of a thread
constexpr int kAhead = 8;                  // tokens of the history that a thread asks for at once
// A token's word: it is in the row's history; it has a bias, and which (9 bits); how often it was generated.
constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u;
constexpr int kHitShift = 21;
constexpr uint32_t kMadeMask = (1u << kHitShift) - 1;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
struct Four {  // four logits of one load: their four results are one 16-byte store, a warp's lie together
  using Raw = uint2;
};
template <>
struct Four<float> {
  using Raw = uint4;
};

template <typename T, bool kAligned>
__global__ void __launch_bounds__(kThreads, 4) process_logits_kernel(const LogitsParams p) {
  __shared__ __align__(16) uint32_t counts[kSlice];
  __shared__ __align__(16) int hit_ids[kThreads + 4];
  __shared__ float hit_values[kThreads];
  __shared__ int warp_hits[kThreads / 32];
  using Raw = typename Four<T>::Raw;
  const int row = blockIdx.y, v0 = blockIdx.x * kSlice, here = min(kSlice, p.vocab - v0);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool with_tokens = p.tokens != nullptr;
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.ld + v0;
  float* y = p.out + (int64_t)row * p.vocab + v0;
  after_previous();
  Raw raw[kEach / 4];
  T single[kAligned ? 1 : kEach];
  if (kAligned) {
#pragma unroll
    for (int u = 0; u < kEach / 4; ++u)
      if ((u * kThreads + tid) * 4 < here) raw[u] = __ldcs(reinterpret_cast<const Raw*>(x) + u * kThreads + tid);
  } else {
#pragma unroll
    for (int u = 0; u < kEach; ++u)
      if (u * kThreads + tid < here) single[u] = x[u * kThreads + tid];
  }
  const uint32_t* allowed = p.allowed != nullptr ? reinterpret_cast<const uint32_t*>(p.allowed) + row * p.allowed_ld + (v0 >> 5) : nullptr;
  uint32_t bits[kAligned ? kEach / 4 : 1];
  if (kAligned) {
#pragma unroll
    for (int u = 0; u < kEach / 4; ++u) {
      const int i = (u * kThreads + tid) * 4;
      bits[u] = allowed != nullptr && i < here ? allowed[i >> 5] >> (i & 31) : 0xffffffffu;
    }
  }
  int b0 = 0, b1 = 0;
  if (p.bias_offsets != nullptr) {
    b0 = max(p.bias_offsets[row], 0);
    b1 = min(p.bias_offsets[row + 1], p.bias_count);
  }
  const int* ids = p.tokens + row * p.tokens_ld;
  int held[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) held[u] = with_tokens && u * kThreads + tid < p.tokens_width ? ids[u * kThreads + tid] : -1;
  int n = 0, prompt = 0;
  if (with_tokens) {
    n = min(p.token_lens != nullptr ? p.token_lens[row] : p.tokens_width, p.tokens_width);
    prompt = p.prompt_lens != nullptr ? p.prompt_lens[row] : 0;
  }
  const float rep = p.repetition != nullptr ? p.repetition[row] : 1.f;
  const float inv_rep = 1.f / rep;  // instead of a quotient a logit: one rounding more
  const float freq = p.frequency != nullptr ? p.frequency[row] : 0.f;
  const float pres = p.presence != nullptr ? p.presence[row] : 0.f;
  const bool counted = with_tokens || b1 > b0;
  int hits = 0;
  if (counted) {
    const int bias_id = b0 + tid < b1 ? p.bias_ids[b0 + tid] - v0 : -1;
    const float bias = b0 + tid < b1 ? p.bias_values[b0 + tid] : 0.f;
    const bool hit = bias_id >= 0 && bias_id < here;
#pragma unroll
    for (int i = 0; i < kEach / 4; ++i) reinterpret_cast<uint4*>(counts)[i * kThreads + tid] = make_uint4(0, 0, 0, 0);
    const uint32_t mask = __ballot_sync(0xffffffffu, hit);
    if (lane == 0) warp_hits[warp] = __popc(mask);
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += warp_hits[w];
      hits += warp_hits[w];
    }
    if (hit) {
      const int k = before + __popc(mask & ((1u << lane) - 1));
      hit_ids[k] = bias_id;
      hit_values[k] = bias;
    }
    if (tid < 4) hit_ids[hits + tid] = -1;
    auto count = [&](int id, int i) {
      const int at = id - v0;
      if (i < n && at >= 0 && at < here) {
        if (i >= prompt) atomicAdd(&counts[at], 1u);
        else atomicOr(&counts[at], kSeen);
      }
    };
#pragma unroll
    for (int u = 0; u < kAhead; ++u) count(held[u], u * kThreads + tid);
#pragma unroll 4
    for (int i = kAhead * kThreads + tid; i < n; i += kThreads) count(ids[i], i);
    if (hits > 0) {
      __syncthreads();
      if (tid < hits) {
        const int id = hit_ids[tid];
        int first = tid, others = 0;
        for (int k = 0; k < hits; k += 4) {
          const int4 h = *reinterpret_cast<const int4*>(hit_ids + k);
          others += (h.x == id) + (h.y == id) + (h.z == id) + (h.w == id);
          if (h.w == id) first = min(first, k + 3);
          if (h.z == id) first = min(first, k + 2);
          if (h.y == id) first = min(first, k + 1);
          if (h.x == id) first = min(first, k);
        }
        if (first == tid) {
          atomicOr(&counts[id], kBiased | (uint32_t)tid << kHitShift);
          if (others > 1) {
            float sum = 0.f;
            for (int k = tid; k < hits; ++k)
              if (hit_ids[k] == id) sum += hit_values[k];
            hit_values[tid] = sum;  // no other thread sums this id
          }
        }
      }
    }
    __syncthreads();
  }
  auto marked = [&](float v, uint32_t c) {
    const uint32_t made = c & kMadeMask;
    if (c & (kSeen | kMadeMask)) v *= v > 0.f ? inv_rep : rep;
    if (made) v -= fmaf(freq, (float)made, pres);
    if (c & kBiased) v += hit_values[c >> kHitShift & (kThreads - 1)];
    return v;
  };
  if (kAligned) {
#pragma unroll
    for (int u = 0; u < kEach / 4; ++u) {
      const int i = (u * kThreads + tid) * 4;
      if (i >= here) break;
      const T* e = reinterpret_cast<const T*>(&raw[u]);
      float v[4] = {to_float(e[0]), to_float(e[1]), to_float(e[2]), to_float(e[3])};
      if (counted) {
        const uint4 c = *reinterpret_cast<const uint4*>(counts + i);
        if (c.x | c.y | c.z | c.w) {
          if (c.x) v[0] = marked(v[0], c.x);
          if (c.y) v[1] = marked(v[1], c.y);
          if (c.z) v[2] = marked(v[2], c.z);
          if (c.w) v[3] = marked(v[3], c.w);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (!(bits[u] >> k & 1)) v[k] = -INFINITY;
      __stcs(reinterpret_cast<float4*>(y + i), make_float4(v[0], v[1], v[2], v[3]));
    }
  } else {
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int i = u * kThreads + tid;
      if (i >= here) break;
      float v = to_float(single[u]);
      if (counted && counts[i]) v = marked(v, counts[i]);
      if (allowed != nullptr && !(allowed[i >> 5] >> (i & 31) & 1)) v = -INFINITY;
      y[i] = v;
    }
  }
  // ---- a row with more biases than threads: kThreads more at a time, added to what has been written
  for (int base = b0 + kThreads; base < b1; base += kThreads) {
    __syncthreads();
    const int many = min(kThreads, b1 - base);
    if (tid < many) {
      hit_ids[tid] = p.bias_ids[base + tid] - v0;
      hit_values[tid] = p.bias_values[base + tid];
    }
    __syncthreads();
    if (tid >= many) continue;
    const int id = hit_ids[tid];
    bool first = id >= 0 && id < here && !(allowed != nullptr && !(allowed[id >> 5] >> (id & 31) & 1));
    for (int k = 0; first && k < tid; ++k) first = hit_ids[k] != id;
    if (first) {
      float sum = 0.f;
      for (int k = tid; k < many; ++k)
        if (hit_ids[k] == id) sum += hit_values[k];
      y[id] += sum;
    }
  }
}

template <typename T>
cudaError_t launch(const LogitsParams& p, cudaStream_t stream) {
  const dim3 grid((unsigned)((p.vocab + kSlice - 1) / kSlice), (unsigned)p.rows);
  // Four logits at a time where every row starts on their boundary, and ends on one.
  const bool aligned = p.vocab % 4 == 0 && p.ld % 4 == 0 && reinterpret_cast<uintptr_t>(p.logits) % (4 * sizeof(T)) == 0 &&
                       reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
  return launch_after_previous(aligned ? process_logits_kernel<T, true> : process_logits_kernel<T, false>, grid, kThreads, 0,
                               stream, p);
}

}  // namespace

namespace mimir {
cudaError_t launch_process_logits(const LogitsParams& p, LogitsType type, cudaStream_t stream) {
  if (type == kLogitsFloat) return launch<float>(p, stream);
  return type == kLogitsHalf ? launch<__half>(p, stream) : launch<__nv_bfloat16>(p, stream);
}
}  // namespace mimir
