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
// before it knows how many count, the biases before it knows which are its own.  It counts the row's
// tokens that fall into its slice in shared memory (whole numbers, so the order of the atomics does not
// matter); a token's word also says which bias is its own, and where an id has several, a warp sums them
// in their order.  The history is read by every block of a row, from L2 after the
// first, so slices are large.
//
// Rows need not start on a boundary of four logits (an odd vocabulary, a view of padded logits): a slice
// starts at the boundary before, and its first and last four may be partly another row's, which are
// neither read nor written.
//
// Measured on B200: 128 rows of 65536 bf16 logits, up to 4000 tokens, 300 biases and a mask each: 16.5 us
// for 53 MB (3.2 TB/s; without tokens, biases and mask 11 us); fp32 21 us; 65535 logits 20 us (one logit at
// a time 39); 65535 of rows of 65536 22 us; one row 5 us, of which its start is most.  Halves or doubles of
// slice and block take 23 and 20 us.
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

// How rows lie: on boundaries of four logits, in and out; as far from one in as out, so that four results are one
// store; or in some other way: results go through shared memory and are stored one by one, a warp's together.
// (fp32 rows of the last two kinds: three blocks an SM, since at four 32 registers spill: 22 us instead of 23.)
enum Rows { kRowsAligned, kRowsAlike, kRowsOther };

template <typename T, Rows kRows>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 && kRows != kRowsAligned ? 3 : 4)
    process_logits_kernel(const LogitsParams p) {
  __shared__ __align__(16) uint32_t counts[kSlice];
  __shared__ int hit_ids[kThreads], again[kThreads];  // a thread's bias; ids that came again
  __shared__ float hit_values[kThreads];
  __shared__ int repeats;
  using Raw = typename Four<T>::Raw;
  const int row = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // The slice: the row's logits v0 + i, lo <= i < here; where i is a multiple of four, they lie on the boundary.
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  const int lead = kRows == kRowsAligned ? 0 : (int)(reinterpret_cast<uintptr_t>(x) / sizeof(T) & 3);
  const int v0 = blockIdx.x * kSlice - lead, here = min(kSlice, p.vocab - v0);
  const int lo = kRows == kRowsAligned ? 0 : blockIdx.x == 0 ? lead : 0;
  if (kRows != kRowsAligned && here <= 0) return;
  const bool with_tokens = p.tokens != nullptr;
  x += v0;
  float* y = p.out + (int64_t)row * p.vocab + v0;
  auto inside = [&](int i) { return i >= lo && i < here; };
  auto all_inside = [&](int i) { return kRows == kRowsAligned ? i < here : i >= lo && i + 4 <= here; };
  after_previous();
  Raw raw[kEach / 4];
#pragma unroll
  for (int u = 0; u < kEach / 4; ++u) {
    const int i = (u * kThreads + tid) * 4;
    if (all_inside(i)) raw[u] = __ldcs(reinterpret_cast<const Raw*>(x + i));
    else if (kRows != kRowsAligned) {
      T* e = reinterpret_cast<T*>(&raw[u]);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (inside(i + k)) e[k] = x[i + k];
    }
  }
  const uint32_t* allowed = p.allowed != nullptr ? reinterpret_cast<const uint32_t*>(p.allowed) + row * p.allowed_ld : nullptr;
  uint32_t bits[kEach / 4];
#pragma unroll
  for (int u = 0; u < kEach / 4; ++u) {
    const int i = (u * kThreads + tid) * 4, v = v0 + i;
    bits[u] = 0xffffffffu;
    if (allowed == nullptr || i >= here) continue;
    if (kRows == kRowsAligned) bits[u] = allowed[v >> 5] >> (v & 31);
    else {  // four bits that may lie in two words
      const uint32_t low = v >= 0 ? allowed[v >> 5] : 0;
      const uint32_t high = (v & 31) > 28 && (v | 31) + 1 < p.vocab ? allowed[(v >> 5) + 1] : 0;
      bits[u] = __funnelshift_r(low, high, v & 31);
    }
  }
  int b0 = 0, b1 = 0;
  if (p.bias_offsets != nullptr) {
    b0 = min(max(p.bias_offsets[row], 0), p.bias_count);  // what is added to it stays in 32 bits
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
  if (counted) {
    const int bias_id = b0 + tid < b1 ? p.bias_ids[b0 + tid] - v0 : 0;
    const float bias = b0 + tid < b1 ? p.bias_values[b0 + tid] : 0.f;
    const bool hit = b0 + tid < b1 && inside(bias_id);
#pragma unroll
    for (int i = 0; i < kEach / 4; ++i) reinterpret_cast<uint4*>(counts)[i * kThreads + tid] = make_uint4(0, 0, 0, 0);
    hit_ids[tid] = hit ? bias_id : -1;
    hit_values[tid] = bias;
    if (tid == 0) repeats = 0;
    __syncthreads();
    if (hit && atomicOr(&counts[bias_id], kBiased | (uint32_t)tid << kHitShift) & kBiased) again[atomicAdd(&repeats, 1)] = bias_id;
    auto count = [&](int id, int i) {
      const int at = id - v0;
      if (i < n && inside(at)) {
        if (i >= prompt) atomicAdd(&counts[at], 1u);
        else atomicOr(&counts[at], kSeen);
      }
    };
#pragma unroll
    for (int u = 0; u < kAhead; ++u) count(held[u], u * kThreads + tid);
#pragma unroll 4
    for (int i = kAhead * kThreads + tid; i < n; i += kThreads) count(ids[i], i);
    __syncthreads();
    // An id with several biases: a warp sums them in their order, and the first one's place holds the sum.
    const int many = repeats;
    for (int r = warp; r < many; r += kThreads / 32) {
      const int id = again[r];
      bool taken = false;
      for (int k = lane; k < r; k += 32) taken |= again[k] == id;
      if (__any_sync(0xffffffffu, taken)) continue;
      int first = -1;
      float sum = 0.f;
      for (int base = 0; base < kThreads; base += 32)
        for (uint32_t m = __ballot_sync(0xffffffffu, hit_ids[base + lane] == id); m; m &= m - 1) {
          const int k = base + __ffs(m) - 1;
          if (first < 0) first = k;
          sum += hit_values[k];
        }
      __syncwarp();
      if (lane == 0) {
        counts[id] = (counts[id] & (kSeen | kMadeMask)) | kBiased | (uint32_t)first << kHitShift;
        hit_values[first] = sum;
      }
    }
    if (many > 0) __syncthreads();
  }
  auto marked = [&](float v, uint32_t c) {
    const uint32_t made = c & kMadeMask;
    if (c & (kSeen | kMadeMask)) v *= v > 0.f ? inv_rep : rep;
    if (made) v -= fmaf(freq, (float)made, pres);
    if (c & kBiased) v += hit_values[c >> kHitShift & (kThreads - 1)];
    return v;
  };
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
    if (kRows == kRowsOther) {
      *reinterpret_cast<float4*>(counts + i) = make_float4(v[0], v[1], v[2], v[3]);
    } else if (all_inside(i)) {
      __stcs(reinterpret_cast<float4*>(y + i), make_float4(v[0], v[1], v[2], v[3]));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (inside(i + k)) y[i + k] = v[k];
    }
  }
  if (kRows == kRowsOther) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kEach; ++u)
      if (inside(u * kThreads + tid)) __stcs(y + u * kThreads + tid, __uint_as_float(counts[u * kThreads + tid]));
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
    bool first = inside(id) && (allowed == nullptr || allowed[(v0 + id) >> 5] >> ((v0 + id) & 31) & 1);
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
  const uintptr_t in = reinterpret_cast<uintptr_t>(p.logits) / sizeof(T) % 4, out = reinterpret_cast<uintptr_t>(p.out) / 4 % 4;
  const bool rows_aligned = p.vocab % 4 == 0 && p.ld % 4 == 0 && in == 0 && out == 0;
  const bool rows_alike = in == out && (p.rows == 1 || p.vocab % 4 == p.ld % 4);
  const dim3 grid((unsigned)((p.vocab + (rows_aligned ? 0 : 3) + kSlice - 1) / kSlice), (unsigned)p.rows);
  return launch_after_previous(rows_aligned ? process_logits_kernel<T, kRowsAligned>
                               : rows_alike ? process_logits_kernel<T, kRowsAlike>
                                            : process_logits_kernel<T, kRowsOther>,
                               grid, kThreads, 0, stream, p);
}

}  // namespace

namespace mimir {
cudaError_t launch_process_logits(const LogitsParams& p, LogitsType type, cudaStream_t stream) {
  if (type == kLogitsFloat) return launch<float>(p, stream);
  return type == kLogitsHalf ? launch<__half>(p, stream) : launch<__nv_bfloat16>(p, stream);
}
}  // namespace mimir
