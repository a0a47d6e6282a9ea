// The 8-bit paged key/value cache: its layout, the checks of its tensors and its status word.
//
//   pages   e4m3  [N, 2, KV, P, 128]   k then v; P tokens a page, a power of two in [16, 256]
//   scales  fp32  [N, 2, KV, P / 16]   a power of two for 16 tokens of one head: value = byte * scale;
//                                      NaN marks a block that was given a value that is not finite
//   table   int32 [S, W]               page of tokens [P*j, P*j + P) of slot s, -1 for none
//   lens    int32 [S]                  tokens of slot s
//   refs    int32 [N]                  how many slots hold a page
#pragma once

#include <c10/util/Exception.h>
#include <torch/extension.h>

namespace mimir {

constexpr int kCacheDim = 128;    // head dimension
constexpr int kCacheBlock = 16;   // tokens that share a scale
constexpr int kCacheMinExp = -32; // smallest scale 2^-32: smaller values round to zero

// Status codes of the cache kernels (the first one since the last read is kept).
enum CacheStatus : int {
  kCacheOk = 0,
  kCacheBadSlot = 1,    // a slot outside the page table
  kCacheBadPage = 2,    // a page that the table does not hold, or one outside the pool
  kCacheBadLength = 3,  // fewer tokens in a slot than new ones, or a position outside the rotary tables
  kCacheTimeout = 4,    // a wait inside a kernel ran out
};

int* cache_status_word(const at::Device& dev);

#define CACHE_CHECK(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

inline void check_int32(const at::Tensor& t, const char* name, int64_t dim, const at::Device& dev) {
  CACHE_CHECK(t.device() == dev && t.scalar_type() == at::kInt && t.dim() == dim && t.is_contiguous(), name,
              " must be a contiguous int32 tensor of ", dim, " dimension(s) on ", dev);
}

// `lead`: dimensions before the page's (0, or 1 for a layer dimension).
inline void check_pool(const at::Tensor& pages, const at::Tensor& scales, int64_t lead) {
  CACHE_CHECK(pages.is_cuda() && pages.scalar_type() == at::kFloat8_e4m3fn && pages.is_contiguous() &&
                  pages.dim() == 5 + lead,
              "pages must be a contiguous float8_e4m3fn CUDA tensor of ", 5 + lead, " dimensions");
  const int64_t P = pages.size(lead + 3);
  CACHE_CHECK(pages.size(lead + 1) == 2 && pages.size(lead + 4) == kCacheDim && pages.size(lead + 2) >= 1,
              "pages must be [pages, 2, kv_heads, page_size, 128]");
  CACHE_CHECK(P >= 16 && P <= 256 && (P & (P - 1)) == 0, "page_size must be 16, 32, 64, 128 or 256, not ", P);
  CACHE_CHECK(reinterpret_cast<uintptr_t>(pages.data_ptr()) % 16 == 0, "pages must start on a 16-byte boundary");
  CACHE_CHECK(scales.device() == pages.device() && scales.scalar_type() == at::kFloat && scales.is_contiguous() &&
                  scales.dim() == 4 + lead,
              "scales must be a contiguous float32 tensor beside the pages");
  for (int64_t i = 0; i < lead + 3; ++i)
    CACHE_CHECK(scales.size(i) == pages.size(i), "scales must be [pages, 2, kv_heads, page_size / 16]");
  CACHE_CHECK(scales.size(lead + 3) == P / kCacheBlock, "scales must be [pages, 2, kv_heads, page_size / 16]");
  CACHE_CHECK(pages.size(lead) * 2 * pages.size(lead + 2) < (int64_t(1) << 31), "the pool has too many pages");
}

// Page table, lengths and the batch: sequence i of the batch is slot seqs[i] and has the rows
// cu_new[i] .. cu_new[i + 1] of the new tokens.
inline void check_batch(const at::Tensor& table, const at::Tensor& lens, const at::Tensor& seqs,
                        const at::Tensor& cu_new, const at::Device& dev) {
  check_int32(table, "page_table", 2, dev);
  check_int32(lens, "seq_lens", 1, dev);
  check_int32(seqs, "seqs", 1, dev);
  check_int32(cu_new, "cu_new", 1, dev);
  CACHE_CHECK(lens.size(0) == table.size(0), "seq_lens needs one length for each row of page_table");
  CACHE_CHECK(cu_new.size(0) == seqs.size(0) + 1, "cu_new needs one more entry than seqs");
}

// Rows [T, heads, 128] of 16-bit values whose last dimension is contiguous and 16-byte aligned.
inline void check_rows(const at::Tensor& x, const char* name, const at::Device& dev) {
  CACHE_CHECK(x.device() == dev && x.dim() == 3 && x.size(2) == kCacheDim && x.stride(2) == 1, name,
              " must be [tokens, heads, 128] on ", dev, " with contiguous heads");
  CACHE_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, name, " must be bfloat16 or float16");
  CACHE_CHECK(reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && x.stride(0) % 8 == 0 && x.stride(1) % 8 == 0, name,
              " must start on a 16-byte boundary in every head");
}

}  // namespace mimir
