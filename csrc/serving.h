// The serving kernels' interface between their device code (kv_cache.cu, cache_attention.cu,
// logits.cu) and the functions that check tensors and launch them (serving.cpp).
//
// The 8-bit paged key/value cache:
//   pages   e4m3  [N, 2, KV, P, 128]   k then v; P tokens a page, a power of two in [16, 256]
//   scales  fp32  [N, 2, KV, P / 16]   a power of two for 16 tokens of one head: value = byte * scale;
//                                      NaN marks a block that was given a value that is not finite
//   table   int32 [S, W]               page of tokens [P*j, P*j + P) of slot s, -1 for none
//   lens    int32 [S]                  tokens of slot s
//   refs    int32 [N]                  how many slots hold a page
// Sequence i of a batch is slot seqs[i] and has the rows cu[i] .. cu[i + 1] of the new tokens, the last
// ones of its slot.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace mimir {

constexpr int kCacheDim = 128;     // head dimension
constexpr int kCacheBlock = 16;    // tokens that share a scale
constexpr int kCacheMinExp = -32;  // smallest scale 2^-32: smaller values round to zero

// Status codes of the cache kernels (the first one since the last read is kept).
enum CacheStatus : int {
  kCacheOk = 0,
  kCacheBadSlot = 1,    // a slot outside the page table
  kCacheBadPage = 2,    // a page that the table does not hold, or one outside the pool
  kCacheBadLength = 3,  // fewer tokens in a slot than new ones, a position outside the rotary tables, or rows
                        // of a sequence outside the call's
  kCacheTimeout = 4,    // a wait inside a kernel ran out
};

// Launches on `stream` so that the kernel is set up while the one before it ends: 1.2 to 2.4 us less a call of
// cache_attention.  The kernel calls after_previous() before it touches global memory: there it waits until
// all that came before is done and visible.  (Letting the next kernel start earlier than at a kernel's end
// cost the larger calls 1 us: its blocks wait where this one's could run.)
template <typename... P, typename... A>
inline cudaError_t launch_after_previous(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                                         const A&... args) {
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, P(args)...);
}
#ifdef __CUDACC__
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Rows cu[i] .. cu[i + 1] of sequence i, as far as the call has them.  Not `good` where they leave its rows or
// run backwards: the sequence is skipped then, its rows become zeros, and kCacheBadLength is reported.  (Bounds
// that run backwards by more than a block of rows may leave rows unwritten in the kernels that search them.)
struct NewRows {
  int first, count;
  bool good;
};
__device__ __forceinline__ NewRows new_rows(const int* cu, int i, int tokens) {
  const int a = cu[i], b = cu[i + 1];
  const int first = min(max(a, 0), tokens);
  return {first, max(min(b, tokens) - first, 0), a >= 0 && a <= b && b <= tokens};
}
// The report, by a block that has no rows of its own.
__device__ __forceinline__ void check_bounds(const int* cu, int n, int tokens, int* status) {
  for (int i = threadIdx.x; i < n; i += blockDim.x)
    if (!new_rows(cu, i, tokens).good) atomicCAS(status, 0, kCacheBadLength);
}
#endif

// ---------------------------------------------------------------- kv_cache.cu
cudaError_t cache_status_address(void** word);  // of the current device

struct AppendParams {
  const void *q, *k, *v;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;  // strides in elements
  void* q_out;                                          // [tokens, H, 128]
  const float *cos, *sin;
  int64_t positions;
  uint8_t* pages;
  float* scales;
  int64_t npages;
  const int *table, *lens, *seqs, *cu;
  int slots, width, n, tokens, H, KV, page;
  int* status;
};
cudaError_t launch_cache_append(const AppendParams& p, bool bf16, cudaStream_t stream);

struct Book {  // page table, lengths and counts
  int *table, *lens, *refs;
  int slots, width, npages, page;
  int* status;
};
constexpr int kBookBatch = 4096;  // sequences of one bookkeeping call
cudaError_t launch_cache_reserve(const Book& b, const int* seqs, const int* counts, int n, int* found, int* missing,
                                 cudaStream_t stream);
cudaError_t launch_cache_free(const Book& b, const int* seqs, int n, cudaStream_t stream);
// from, to: [n]; found: [n]
cudaError_t launch_cache_fork(const Book& b, const int* src, const int* dst, int n, int* from, int* to, int* found,
                              int* missing, cudaStream_t stream);
// to, holes: [npages]
cudaError_t launch_cache_plan(const int* refs, int npages, int* out_refs, int room, int* holes, int* to, int* kept,
                              int* missing, cudaStream_t stream);

// Copies page from[i] of every layer to page to[i] (i itself where `from` is null; nothing where either is
// negative or both are the same page of one pool), bytes and scales, unless *missing is not zero.
struct CopyParams {
  const uint8_t* pages;
  const float* scales;
  uint8_t* out_pages;
  float* out_scales;
  int64_t npages, out_npages, page_bytes;
  int scale_floats, layers, n;
  const int *from, *to, *missing;
  int* status;
  // compaction: every entry of the page table becomes to[entry]
  const int* table;
  int* out_table;
  int64_t entries;
};
cudaError_t launch_cache_copy(const CopyParams& p, cudaStream_t stream);

// ---------------------------------------------------------------- cache_attention.cu
constexpr int kAttentionKeys = 64;         // keys of a unit
constexpr int kAttentionRows = 16;         // query rows of a tile, at most (the kernel for few rows has 8)
constexpr int kAttentionSeqs = 1024;       // sequences of one launch
constexpr int kAttentionBlocks = 3 * 148;  // at most three blocks an SM
// A segment's ends (queries in, results out) take as long as some five units of keys: its share of
// the line of work is that much longer, or blocks with many short segments would finish last.
constexpr int kAttentionEnds = 5;

struct AttentionParams {
  const void* q;
  int64_t q_tok, q_head;
  void* out;            // [tokens, H, 128]
  const float* scales;
  const int *table, *lens, *seqs, *cu, *prefix;
  int slots, width, n, tokens, H, KV, group, page, page_shift, npages;
  float scale_log2;
  int* arrived;         // per block: parts of the segment that it begins, zero between calls
  float* parts;         // [blocks][2][rows of a tile][128]
  float2* part_ml;      // [blocks][2][rows of a tile]: maximum and sum
  float join_cost;      // four times the segments that the sequences have, about
  int first_batch;      // the call's first launch: rows before all sequences become zeros
  int last_batch;       // its last launch: those after all sequences do
  int* status;
};
cudaError_t launch_cache_attention(const CUtensorMap& map, const AttentionParams& p, bool bf16, bool full, int grid,
                                   cudaStream_t stream);

// ---------------------------------------------------------------- cache_prompt.cu
constexpr int kPromptKeys = 128;  // keys of a tile: the box of the map of the pages
// map_q: [tokens, H, 128] with boxes of 128 / group tokens, `group` heads and 64 dimensions.
cudaError_t launch_cache_prompt(const CUtensorMap& map_q, const CUtensorMap& map_pages, const AttentionParams& p, bool bf16,
                                cudaStream_t stream);

// ---------------------------------------------------------------- logits.cu
enum LogitsType { kLogitsFloat, kLogitsHalf, kLogitsBFloat16 };
struct LogitsParams {
  const void* logits;
  int64_t ld;
  float* out;
  int rows, vocab;
  const int *tokens, *token_lens, *prompt_lens;
  int64_t tokens_ld;
  int tokens_width;
  const float *repetition, *presence, *frequency;
  const int *bias_offsets, *bias_ids;
  const float* bias_values;
  int bias_count;
  const int* allowed;
  int64_t allowed_ld;
};
cudaError_t launch_process_logits(const LogitsParams& p, LogitsType type, cudaStream_t stream);

}  // namespace mimir
